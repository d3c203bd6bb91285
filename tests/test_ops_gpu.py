"""The 8-bit operators (vosk.ops) against plain 64-bit forms (int8_ref.py).

Codes, scales and row maps have to be equal.  The product's tolerance counts
its roundings: an integer sum to 32-bit float and an fma for each tap, the
column scale, and up to six more in the epilogue, each half a unit in the last
place (2^-24) of a partial result no larger than the sum of the magnitudes;
then the rounding to the output's type (finfo.eps / 2)."""
import numpy as np
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from vosk import ops
    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _np(t):
    return t.detach().double().cpu().numpy()


def _same_codes(codes, scales, x):
    want_c, want_s = ref.codes_of(_np(x))
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    np.testing.assert_array_equal(codes.cpu().numpy()[:, :want_c.shape[1]], want_c)


# ---- rows to codes


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 512), (3, 63), (5, 64), (4, 65), (257, 96), (33, 1000), (9, 2047), (7, 2049),
                                 (2, 8191), (3, 9000), (1, 40001), (0, 12)])
def test_quantize_rows(ops, t, m, k):
    g = _gen(m * 1000 + k)
    x = (_randn(g, m, k) * torch.exp(2 * _randn(g, m, 1))).to(TYPES[t])
    codes, scales = ops.quantize_rows(x)
    assert codes.shape == (m, ref.pad(k)) and scales.shape == (m,)
    _same_codes(codes, scales, x)


@pytest.mark.parametrize("t", TYPES)
def test_quantize_rows_at_the_edges(ops, t):
    """Halves between codes, zeros, Inf, NaN, subnormals, the type's largest."""
    dt = TYPES[t]
    f = torch.finfo(dt)
    k = 300
    g = _gen(1)
    x = _randn(g, 16, k)
    x[0] = torch.randint(-253, 254, (k,), generator=g, device="cuda") * 0.5
    x[0, 7] = 127  # scale 1: every value a whole code or half way between two
    x[1] = x[0] * 2.0 ** -10
    x[2] = 0
    x[3] = -0.0
    x[4, 299] = float("inf")
    x[5, 0] = float("nan")
    x[6, 100] = -float("inf")
    x[7] = 0
    x[7, 150] = -3.0
    x[8] = f.max * torch.where(x[8] < 0, -1.0, 1.0)
    x[9] = f.max * torch.rand(k, generator=g, device="cuda").clamp(max=0.9)
    x = x.to(dt)
    tiny = f.smallest_normal * f.eps  # the smallest subnormal
    for i, top in ((10, 1), (11, 63), (12, 64), (13, 100), (14, 1000)):
        x[i] = (torch.randint(-top, top + 1, (k,), generator=g, device="cuda").double() * tiny).to(dt)
        x[i, 3] = tiny * top
    x[15] = (f.smallest_normal * x[15].double()).to(dt)
    codes, scales = ops.quantize_rows(x)
    _same_codes(codes, scales, x)
    assert scales[2] == 0 and scales[3] == 0 and torch.isnan(scales[4:7]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k,ld,start", [(33, 37, 1), (512, 515, 3), (130, 1024, 0), (8, 8, 5)])
def test_quantize_rows_strides_and_alignments(ops, t, k, ld, start):
    g = _gen(k)
    flat = _randn(g, 21 * ld + start).to(TYPES[t])
    x = flat[start:start + 20 * ld].view(20, ld)[:, :k]
    codes = torch.full((20, ref.pad(k) + 16), 9, dtype=torch.int8, device="cuda")
    scales = torch.zeros(20, device="cuda")
    out = ops.quantize_rows(x, codes, scales)
    assert out[0] is codes and out[1] is scales
    _same_codes(codes, scales, x)
    assert (codes[:, ref.pad(k):] == 9).all()


def test_quantize_rows_every_second_row_and_row_stride_zero(ops):
    x = _randn(_gen(3), 10, 70)
    _same_codes(*ops.quantize_rows(x[::2]), x[::2])
    with pytest.raises(ValueError, match="overlap"):
        ops.quantize_rows(x[:1].expand(5, 70))
    with pytest.raises(ValueError, match="contiguous"):
        ops.quantize_rows(x.t())


def test_quantize_rows_into_a_cache(ops):
    g = _gen(5)
    x = _randn(g, 50, 96)
    rows = torch.randperm(200, generator=g, device="cuda")[:50].int()
    rows[3], rows[4], rows[5], rows[6] = -1, -7, 200, 2**31 - 1
    codes = torch.full((200, 128), 9, dtype=torch.int8, device="cuda")
    scales = torch.full((200,), -1.0, device="cuda")
    ops.quantize_rows(x, codes, scales, rows=rows)
    want_c, want_s = np.full((200, 128), 9, np.int8), np.full(200, -1, np.float32)
    c, s = ref.codes_of(_np(x))
    for i, to in enumerate(rows.tolist()):
        if 0 <= to < 200:
            want_c[to], want_s[to] = c[i], s[i]
    np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)


def test_quantize_rows_from_rows(ops):
    """Rows gathered from a ring and scattered into a cache through columns of one map."""
    g = _gen(15)
    x = _randn(g, 300, 96)
    both = torch.stack([torch.randint(0, 300, (70,), generator=g, device="cuda"), torch.randperm(200, generator=g, device="cuda")[:70]], 1).int()
    both[3, 0], both[4, 0], both[5, 1] = -1, 300, 200
    codes = torch.full((200, 128), 9, dtype=torch.int8, device="cuda")
    scales = torch.full((200,), -1.0, device="cuda")
    ops.quantize_rows(x, codes, scales, rows=both[:, 1], from_rows=both[:, 0])
    want_c, want_s = np.full((200, 128), 9, np.int8), np.full(200, -1, np.float32)
    c, s = ref.codes_of(_np(x))
    for fr, to in both.tolist():
        if 0 <= fr < 300 and 0 <= to < 200:
            want_c[to], want_s[to] = c[fr], s[fr]
    np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)


@pytest.mark.parametrize("count", [-2, 0, 1, 7, 20, 99])
def test_quantize_rows_leaves_rows_past_the_count(ops, count):
    x = _randn(_gen(8), 20, 70)
    codes = torch.full((20, 128), 9, dtype=torch.int8, device="cuda")
    scales = torch.full((20,), -1.0, device="cuda")
    ops.quantize_rows(x, codes, scales, count=torch.tensor([count], dtype=torch.int32, device="cuda"))
    n = max(0, min(20, count))
    _same_codes(codes[:n], scales[:n], x[:n])
    assert (codes[n:] == 9).all() and (scales[n:] == -1).all()


def test_quantize_rows_offsets_past_32_bits(ops):
    """Rows of x 2^30 elements apart, code rows at the end of a cache of over 4 GiB."""
    flat = torch.empty(3 * 2**30 + 100, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((4, 100), (2**30, 1))
    x.copy_(_randn(_gen(6), 4, 100))
    n = 2**32 // 128 + 10
    codes = torch.empty(n, 128, dtype=torch.int8, device="cuda")
    scales = torch.empty(n, device="cuda")
    rows = torch.tensor([n - 1, 0, n - 2, n // 2 + 1], dtype=torch.int32, device="cuda")
    ops.quantize_rows(x, codes, scales, rows=rows)
    _same_codes(codes[rows.long()], scales[rows.long()], x)


def test_quantize_weight(ops):
    w = _randn(_gen(7), 20, 2 * 40)
    codes, scales = ops.quantize_weight(w, taps=2)
    c, s = ref.codes_of(_np(w))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    got = codes.view(20, 2, 64).cpu().numpy()
    np.testing.assert_array_equal(got[:, :, :40].reshape(20, 80), c[:, :80])
    assert (got[:, :, 40:] == 0).all()


# ---- row maps


def _map_case(ops, streams, most, taps, step, page, pages, limits, clamp, seed, extra=5, first_lo=-50, first_hi=5000):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, most + 1, streams).astype(np.int32)
    lengths[rng.random(streams) < 0.1] = 0
    lengths[rng.random(streams) < 0.05] = -3
    first = rng.integers(first_lo, first_hi, streams).astype(np.int32)
    table = rng.permutation(streams * pages).astype(np.int32).reshape(streams, pages)
    table[rng.random(table.shape) < 0.05] = -1
    low = high = None
    if limits:
        low = (first - rng.integers(0, 6, streams)).astype(np.int32)
        high = (first + lengths + rng.integers(-4, 4, streams)).astype(np.int32)
    offsets = [int(v) for v in rng.integers(-7, 8, taps)]
    total = int(sum(-(-max(int(v), 0) // step) for v in lengths))
    before = np.full((max(0, total + extra), taps), -9, np.int32)
    dev = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    rows = dev(before)
    starts, got = ops.frame_map(dev(lengths), dev(first), dev(table), page, rows, offsets=offsets, step=step, low=dev(low),
                                high=dev(high), clamp=clamp)
    assert got is rows
    want_s, want_r = ref.frame_map(lengths, first, table, page, offsets, step, low, high, clamp, before)
    np.testing.assert_array_equal(starts.cpu().numpy(), want_s)
    np.testing.assert_array_equal(rows.cpu().numpy(), want_r)


@pytest.mark.parametrize("limits,clamp", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("streams,most,taps,step,page,pages", [
    (1, 1, 1, 1, 1, 1), (1, 51, 3, 1, 512, 1), (3, 7, 2, 3, 16, 2), (40, 60, 5, 2, 7, 5), (256, 51, 3, 3, 512, 1),
    (300, 20, 16, 1, 4, 3), (5, 700, 2, 1, 64, 8), (1023, 9, 1, 1, 100, 1), (4097, 3, 2, 1, 16, 1), (9000, 4, 1, 2, 8, 2)])
def test_frame_map(ops, streams, most, taps, step, page, pages, limits, clamp):
    _map_case(ops, streams, most, taps, step, page, pages, limits, clamp, streams + most)


@pytest.mark.parametrize("clamp", [False, True])
@pytest.mark.parametrize("only", ["low", "high"])
def test_frame_map_one_limit(ops, only, clamp):
    rng = np.random.default_rng(7)
    lengths, first = rng.integers(0, 20, 30).astype(np.int32), rng.integers(-20, 20, 30).astype(np.int32)
    limit = (first + rng.integers(0, 10, 30)).astype(np.int32)
    table = rng.permutation(60).astype(np.int32).reshape(30, 2)
    before = np.full((int(lengths.sum()), 3), -9, np.int32)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    rows = dev(before)
    ops.frame_map(dev(lengths), dev(first), dev(table), 16, rows, offsets=(-5, 0, 6), clamp=clamp, **{only: dev(limit)})
    kw = dict(low=None, high=None)
    kw[only] = limit
    np.testing.assert_array_equal(rows.cpu().numpy(), ref.frame_map(lengths, first, table, 16, (-5, 0, 6), 1, kw["low"], kw["high"], clamp, before)[1])


@pytest.mark.parametrize("off", [2**31 - 1, 2**30 + 5, -2**30 - 3, -2**31])
def test_frame_map_far_offsets(ops, off):
    """Times and offsets whose sums need more than 32 bits, or nearly."""
    first = np.array([0, 5, 2**30 - 3, -2**30, 2**31 - 30, -2**31], np.int32)
    lengths = np.array([4, 7, 9, 3, 11, 5], np.int32)
    table = np.arange(12, dtype=np.int32).reshape(6, 2)[::-1].copy()
    before = np.full((39, 2), -9, np.int32)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    rows = dev(before)
    ops.frame_map(dev(lengths), dev(first), dev(table), 37, rows, offsets=(off, -1))
    np.testing.assert_array_equal(rows.cpu().numpy(), ref.frame_map(lengths, first, table, 37, (off, -1), 1, None, None, True, before)[1])


def test_frame_map_of_a_ring_with_streams_side_by_side(ops):
    """page_stride 1, frame_stride = streams: row (t mod ring) * streams + slot."""
    lengths, first, slots = [3, 5, 2], [60, -3, 7], [2, 0, 5]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.full((10, 2), -9, dtype=torch.int32, device="cuda")
    ops.frame_map(i32(lengths), i32(first), i32(slots).view(3, 1), 64, rows, offsets=(0, 3), strides=(1, 6))
    want = [[((f + i + o) % 64) * 6 + s for o in (0, 3)] for n, f, s in zip(lengths, first, slots) for i in range(n)]
    assert rows.tolist() == want


def test_frame_map_with_less_room_than_rows(ops):
    _map_case(ops, 20, 30, 3, 1, 64, 1, True, True, 2, extra=-40)
    _map_case(ops, 20, 30, 3, 1, 64, 1, True, True, 3, extra=-100000)


def test_frame_map_at_the_ends_of_time(ops):
    """Frame times next to +-2^31: entries outside 32 bits are absent."""
    _map_case(ops, 6, 20, 3, 1, 64, 1, False, True, 4, first_lo=2**31 - 12, first_hi=2**31 - 1)
    _map_case(ops, 6, 20, 3, 1, 64, 1, False, True, 5, first_lo=-2**31, first_hi=-2**31 + 10)


def test_frame_map_no_streams_and_empty_streams(ops):
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rows = torch.full((4, 1), -9, dtype=torch.int32, device="cuda")
    starts, _ = ops.frame_map(none, none, none.view(0, 1), 8, rows)
    assert starts.tolist() == [0] and (rows == -9).all()
    z = torch.zeros(5, dtype=torch.int32, device="cuda")
    starts, _ = ops.frame_map(z, z, z.view(5, 1), 8, rows)
    assert starts.tolist() == [0] * 6 and (rows == -9).all()


def test_frame_map_one_long_stream(ops):
    """A stream longer than its ring: the frames that the ring no longer holds have no row."""
    lengths = torch.tensor([100000], dtype=torch.int32, device="cuda")
    first = torch.tensor([17], dtype=torch.int32, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    rows = torch.full((100000, 1), -9, dtype=torch.int32, device="cuda")
    ops.frame_map(lengths, first, table, 25, rows)
    t = torch.arange(17, 100017)
    want = torch.where(t > 100016 - 100, t % 100, torch.full_like(t, -1))
    assert torch.equal(rows[:, 0].cpu().long(), want)


# ---- the product


def _check(got, v, size, taps, out_type):
    t = TYPES[out_type]
    tol = (2 * taps + 8) * 2.0 ** -24 * size
    tol = tol + torch.finfo(t).eps / 2 * (np.abs(v) + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    got = _np(got)
    assert got.shape == v.shape
    bad = ~(np.abs(got - v) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], v[bad][:5])


def _linear_case(ops, m, n, k, taps, t, out_type, epilogue, seed, cache=None, count=None, given=False):
    """One product; cache: rows of a frame cache read through a map, else float rows in."""
    g = _gen(seed)
    w, ws = ops.quantize_weight(_randn(g, n, taps * k) / (taps * k) ** 0.5, taps)
    e = {}
    if "b" in epilogue:
        e["bias"] = _randn(g, n)
    if "r" in epilogue:
        e["relu"] = True
    if "g" in epilogue:
        e["gain"], e["shift"] = 0.5 + torch.rand(n, generator=g, device="cuda"), _randn(g, n)
    if "s" in epilogue:
        e["residual"], e["residual_scale"] = _randn(g, m, n).to(TYPES[t]), 0.66
    out = torch.full((m, n), 7.0, dtype=TYPES[out_type], device="cuda") if given or count is not None else None
    kw = dict(e, out=out, dtype=TYPES[out_type])
    cnt = None if count is None else torch.tensor([count], dtype=torch.int32, device="cuda")
    rows = None
    if cache is None:
        x = (_randn(g, m, k) * torch.exp(_randn(g, m, 1))).to(TYPES[t])
        got = ops.linear_int8(x, w, ws, count=cnt, **kw)
        codes, scales = ref.codes_of(_np(x))
    else:
        c, s = ops.quantize_rows(_randn(g, cache, k).to(TYPES[t]))
        rows = torch.randint(-1, cache, (m, taps), generator=g, device="cuda", dtype=torch.int32)
        if m > 2:
            rows[1] = -1                     # nothing but the epilogue
            rows[2, 0] = cache               # outside: adds nothing
        got = ops.linear_int8(c, w, ws, scale=s, rows=rows, count=cnt, **kw)
        codes, scales = c.cpu().numpy(), s.cpu().numpy()
    ne = {a: (_np(b) if isinstance(b, torch.Tensor) else b) for a, b in e.items()}
    v, size = ref.linear(codes, scales, None if rows is None else rows.cpu().numpy(), w.cpu().numpy(), ws.cpu().numpy(), taps, **ne)
    used = m if count is None else max(0, min(m, count))
    _check(got[:used], v[:used], size[:used], taps, out_type)
    if count is not None:
        assert (got[used:] == 7.0).all()


SIZES = [(1, 1, 1), (1, 512, 512), (1, 2000, 192), (2, 33, 65), (3, 96, 1024), (7, 777, 1000), (8, 128, 4096), (13, 100, 130), (16, 512, 512),
         (17, 2000, 192), (31, 31, 31), (32, 64, 64), (33, 65, 129), (64, 96, 96), (65, 1001, 257), (100, 100, 100), (127, 128, 128),
         (129, 127, 640), (255, 257, 512), (300, 520, 1536), (513, 192, 100), (1000, 96, 512)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("t,out_type", [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp32")])
def test_linear_float_rows(ops, m, n, k, t, out_type):
    _linear_case(ops, m, n, k, 1, t, out_type, "", m + n + k)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("taps,out_type,epilogue", [(1, "fp32", ""), (2, "fp16", "brgs"), (3, "fp32", "brgs"), (5, "bf16", "bs")])
def test_linear_spliced_rows(ops, m, n, k, taps, out_type, epilogue):
    _linear_case(ops, m, n, k, taps, "fp32", out_type, epilogue, m + n + k + taps, cache=77)


@pytest.mark.parametrize("epilogue", ["", "b", "r", "g", "s", "br", "bg", "rg", "rs", "gs", "brgs"])
@pytest.mark.parametrize("m", [3, 70, 600])
def test_linear_epilogues(ops, m, epilogue):
    for t in TYPES:
        _linear_case(ops, m, 200, 96, 1, t, t, epilogue, m)


@pytest.mark.parametrize("m,count", [(5, 0), (5, 3), (40, 33), (300, 129), (300, 300), (300, 1000), (300, -4), (1030, 1)])
def test_linear_leaves_rows_past_the_count(ops, m, count):
    _linear_case(ops, m, 150, 128, 2, "fp32", "fp32", "brgs", m, cache=50, count=count)
    _linear_case(ops, m, 150, 128, 1, "fp32", "bf16", "b", m, count=count)


@pytest.mark.parametrize("m", [1, 40, 700])
def test_linear_largest_sums_and_nan_rows(ops, m):
    """Codes all +-127 over the longest row allowed; a NaN scale makes its rows NaN and no other."""
    k = 1 << 17
    c = torch.full((3, k), 127, dtype=torch.int8, device="cuda")
    c[1] = -127
    s = torch.tensor([1.0, 0.5, float("nan")], device="cuda")
    w = torch.full((5, k), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    w[2, 1:] = 0
    rows = (torch.arange(m, device="cuda", dtype=torch.int32) % 3).view(m, 1)
    got = _np(ops.linear_int8(c, w, torch.ones(5, device="cuda"), scale=s, rows=rows))
    full = 127.0 * 127 * k
    want = np.array([[full, -full, 127 * 127, full, full]])
    want = np.concatenate([want, -0.5 * want, want * np.nan])[np.arange(m) % 3]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_allclose(got, want, rtol=2.0 ** -24, equal_nan=True)


@pytest.mark.parametrize("m", [4, 100])
def test_linear_strides_and_in_place_residual(ops, m):
    g = _gen(m)
    x = _randn(g, m, 3, 100)[:, 1]                       # rows 300 apart
    w, ws = ops.quantize_weight(_randn(g, 60, 100))
    wide = torch.zeros(60, 256, dtype=torch.int8, device="cuda")
    wide[:, 64:192] = w
    buf = _randn(g, m, 90).half()
    before = buf.clone()
    out = buf[:, 10:70]
    got = ops.linear_int8(x, wide[:, 64:192], ws, residual=out, residual_scale=-2.0, out=out)
    assert got is out
    codes, scales = ref.codes_of(_np(x))
    v, size = ref.linear(codes, scales, None, w.cpu().numpy(), ws.cpu().numpy(), 1, residual=_np(before[:, 10:70]), residual_scale=-2.0)
    _check(out, v, size, 1, "fp16")
    assert torch.equal(buf[:, :10], before[:, :10]) and torch.equal(buf[:, 70:], before[:, 70:])


def test_linear_overflow_and_nan_reach_the_output(ops):
    x = torch.full((40, 64), 6e4, device="cuda")
    w, ws = ops.quantize_weight(torch.ones(33, 64, device="cuda"))
    assert torch.isinf(ops.linear_int8(x, w, ws, dtype=torch.float16)).all()
    bias = torch.zeros(33, device="cuda")
    bias[5] = float("nan")
    y = ops.linear_int8(x, w, ws, bias=bias, relu=True, dtype=torch.bfloat16)
    assert torch.isnan(y[:, 5]).all() and not torch.isnan(y[:, 6:]).any()


def test_linear_cache_offsets_past_32_bits(ops):
    n = 2**32 // 64 + 10
    codes = torch.empty(n, 64, dtype=torch.int8, device="cuda")
    scales = torch.empty(n, device="cuda")
    rows = torch.tensor([[n - 1], [0], [n // 2 + 3], [-1], [n]], dtype=torch.int32, device="cuda").repeat(30, 1)
    at = torch.tensor([n - 1, 0, n // 2 + 3], device="cuda")
    g = _gen(9)
    codes[at] = torch.randint(-127, 128, (3, 64), generator=g, device="cuda", dtype=torch.int8)
    scales[at] = torch.rand(3, generator=g, device="cuda")
    w, ws = ops.quantize_weight(_randn(g, 50, 64))
    small = torch.tensor([[0], [1], [2], [-1], [-1]]).repeat(30, 1).numpy()
    v, size = ref.linear(codes[at].cpu().numpy(), scales[at].cpu().numpy(), small, w.cpu().numpy(), ws.cpu().numpy(), 1)
    _check(ops.linear_int8(codes, w, ws, scale=scales, rows=rows), v, size, 1, "fp32")
    _check(ops.linear_int8(codes, w, ws, scale=scales, rows=rows[:5].contiguous()), v[:5], size[:5], 1, "fp32")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k,taps", [(5, 40, 64, 1), (20, 100, 130, 3), (90, 70, 96, 2), (300, 513, 192, 1), (3000, 2000, 96, 2),
                                        (2100, 2050, 2100, 1)])
def test_linear_mapped_rows(ops, m, n, k, taps, t):
    """Rows read, residual rows and output rows all through one map, as a layer over frame rings has them."""
    g = _gen(m + n)
    c, s = ops.quantize_rows(_randn(g, 99, k))
    w, ws = ops.quantize_weight(_randn(g, n, taps * k) / (taps * k) ** 0.5, taps)
    res = _randn(g, 80, n).to(TYPES[t])
    rows = torch.randint(-1, 100, (m, taps + 2), generator=g, device="cuda", dtype=torch.int32)
    rows[:, taps] = torch.randperm(m + 50, generator=g, device="cuda")[:m].int() - 20    # some outside out
    rows[:, taps + 1] = torch.randint(-1, 82, (m,), generator=g, device="cuda")          # some outside residual
    bias = _randn(g, n)
    out = torch.full((m, n), 7.0, dtype=TYPES[t], device="cuda")
    count = torch.tensor([m - 2], dtype=torch.int32, device="cuda")
    ops.linear_int8(c, w, ws, scale=s, rows=rows[:, :taps], count=count, bias=bias, relu=True, residual=res, residual_scale=0.75, out=out,
                    out_rows=rows[:, taps], residual_rows=rows[:, taps + 1])
    r = rows.cpu().numpy()[:m - 2]
    rf = r[:, taps + 1]
    z = np.where(((rf >= 0) & (rf < 80))[:, None], _np(res)[np.clip(rf, 0, 79)], 0.0)
    v, size = ref.linear(c.cpu().numpy(), s.cpu().numpy(), r[:, :taps], w.cpu().numpy(), ws.cpu().numpy(), taps, bias=_np(bias), relu=True,
                         residual=z, residual_scale=0.75)
    to = r[:, taps]
    ok = (to >= 0) & (to < m)
    _check(out[torch.from_numpy(to[ok]).long().cuda()], v[ok], size[ok], taps, t)
    rest = np.setdiff1d(np.arange(m), to[ok])
    assert (out[torch.from_numpy(rest).cuda()] == 7.0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k,taps", [(1, 17, 5, 1), (1, 96, 512, 2), (17, 96, 512, 2), (17, 512, 96, 2), (32, 40, 100, 3), (9, 50, 64, 16), (3, 33, 4096, 2),
                                        (33, 40, 100, 3), (300, 96, 512, 2)])
def test_linear_float_rows_through_a_map(ops, m, n, k, taps, t):
    """Quantised in the call or beforehand: the same bits; absent rows, one row under several taps."""
    g = _gen(m + n + k)
    x = (_randn(g, 50, k) * torch.exp(_randn(g, 50, 1))).to(TYPES[t])
    x[7] = 0
    x[8, 0] = float("inf")
    w, ws = ops.quantize_weight(_randn(g, n, taps * k) / (taps * k) ** 0.5, taps)
    rows = torch.randint(-1, 51, (m, taps), generator=g, device="cuda", dtype=torch.int32)
    rows[0] = 3
    if m > 2:
        rows[1], rows[2, 0] = -1, 7
    c, s = ops.quantize_rows(x)
    want = ops.linear_int8(c, w, ws, scale=s, rows=rows)
    got = ops.linear_int8(x, w, ws, rows=rows)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    fine = ~(rows == 8).any(1)
    assert not torch.isnan(got[fine]).any() and torch.isnan(got[~fine]).all()
    v, size = ref.linear(*(a[:len(a)] for a in ref.codes_of(np.where(np.isfinite(_np(x)), _np(x), 0))), rows.cpu().numpy(), w.cpu().numpy(), ws.cpu().numpy(), taps)
    f = fine.cpu().numpy()
    _check(got[fine], v[f], size[f], taps, "fp32")


def test_linear_empty(ops):
    w, ws = ops.quantize_weight(torch.ones(3, 64, device="cuda"))
    assert ops.linear_int8(torch.ones(0, 64, device="cuda"), w, ws).shape == (0, 3)
    assert ops.linear_int8(torch.ones(2, 64, device="cuda"), w[:0], ws[:0]).shape == (2, 0)


def test_refusals(ops):
    g = _gen(0)
    x = _randn(g, 4, 100)
    c, s = ops.quantize_rows(x)
    w, ws = ops.quantize_weight(_randn(g, 8, 100))
    rows = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    cases = [
        (lambda: ops.quantize_rows(x.double()), "float32"),
        (lambda: ops.quantize_rows(x.clone().requires_grad_()), "gradient"),
        (lambda: ops.quantize_rows(x, c), "together"),
        (lambda: ops.quantize_rows(x, rows=rows[:, 0]), "codes and scales"),
        (lambda: ops.quantize_rows(x, c[:, :64], s), "columns"),
        (lambda: ops.quantize_rows(x, c[:3], s[:3]), "fewer"),
        (lambda: ops.quantize_rows(x, c, s, rows=rows[:3, 0]), "4 elements"),
        (lambda: ops.quantize_rows(x[:, :0]), "columns"),
        (lambda: ops.linear_int8(c, w, ws), "scales"),
        (lambda: ops.linear_int8(c[:, :100], w, ws, scale=s), "multiple"),
        (lambda: ops.linear_int8(c, w[:, :64], ws, scale=s), "columns"),
        (lambda: ops.linear_int8(c, w, ws[:3], scale=s), "elements"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, rows=rows.long()), "int32"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, rows=rows.expand(4, 2)), "contiguous"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, out_rows=rows[:, 0]), "needs an out"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, residual_rows=rows[:, 0]), "needs a residual"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, out=x[:, :8], out_rows=rows[:3, 0]), "elements"),
        (lambda: ops.quantize_rows(x, from_rows=rows[:, 0]), "codes and scales"),
        (lambda: ops.quantize_rows(x, c, s, rows=rows[:3, 0], from_rows=rows[:, 0]), "elements"),
        (lambda: ops.linear_int8(x, w, ws, scale=s), "belongs to codes"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, gain=ws), "together"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, bias=ws.cpu()), "another device"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, residual=x), "residual"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, out=x), "out has"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, dtype=torch.float64), "dtype"),
        (lambda: ops.linear_int8(c, w, None, scale=s), "null"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, bias=3.0), "tensor"),
        (lambda: ops.linear_int8(c, None, ws, scale=s), "tensor"),
        (lambda: ops.linear_int8(x, w, ws, bias=ws.clone().requires_grad_()), "gradient"),
        (lambda: ops.frame_map(rows[:, 0], None, rows, 8, rows), "first"),
        (lambda: ops.frame_map(rows[:, 0], rows[:, 0], rows, 8, rows, offsets=(2**31,)), "32-bit"),
        (lambda: ops.linear_int8(c, w, ws, scale=s, count=rows[:2, 0]), "elements"),
        (lambda: ops.frame_map(rows[:, 0], rows[:3, 0], rows, 8, rows), "elements"),
        (lambda: ops.frame_map(rows[:, 0], rows[:, 0], rows[:2], 8, rows), "row for each"),
        (lambda: ops.frame_map(rows[:, 0], rows[:, 0], rows, 8, rows, offsets=(1, 2)), "contiguous"),
        (lambda: ops.frame_map(rows[:, 0], rows[:, 0], rows, 0, rows), "pages"),
        (lambda: ops.frame_map(rows[:, 0], rows[:, 0], rows, 8, rows, step=0), "step"),
    ]
    for i, (call, what) in enumerate(cases):
        with pytest.raises(ValueError, match=what):
            call()
            pytest.fail(f"case {i} was not refused")


# ---- together


def _layer_inputs(g, streams, frames, dim):
    x = _randn(g, streams * frames, dim)
    lengths = torch.full((streams,), frames, dtype=torch.int32, device="cuda")
    lengths[1] = frames - 4
    return x, lengths


class _Layer:
    """Two spliced layers over frame caches, as a streaming program runs them:
    write the new frames, map, hidden -> bottleneck, write, map, bottleneck ->
    hidden with ReLU, BatchNorm and the bypass."""

    def __init__(self, ops, g, streams, frames, dim, low):
        self.ops, self.streams, self.frames, self.dim = ops, streams, frames, dim
        self.ring = 64
        self.table = torch.arange(streams, dtype=torch.int32, device="cuda").view(streams, 1)
        self.w1, self.s1 = ops.quantize_weight(_randn(g, low, 2 * dim) / (2 * dim) ** 0.5, 2)
        self.w2, self.s2 = ops.quantize_weight(_randn(g, dim, 2 * low) / (2 * low) ** 0.5, 2)
        self.bias, self.gain, self.shift = _randn(g, dim), 0.5 + torch.rand(dim, generator=g, device="cuda"), _randn(g, dim)
        n, i32 = streams * frames, dict(dtype=torch.int32, device="cuda")
        self.c = [torch.zeros(streams * self.ring, ref.pad(d), dtype=torch.int8, device="cuda") for d in (dim, low)]
        self.s = [torch.zeros(streams * self.ring, device="cuda") for _ in range(2)]
        self.write, self.read = torch.full((n, 1), -1, **i32), [torch.full((n, 2), -1, **i32) for _ in range(2)]
        self.starts = [torch.zeros(streams + 1, **i32) for _ in range(3)]
        self.low = torch.zeros(n, low, device="cuda")
        self.out = torch.zeros(n, dim, device="cuda")

    def step(self, x, lengths, first, zero, last):
        o = self.ops
        o.frame_map(lengths, first, self.table, self.ring, self.write, self.starts[0])
        o.quantize_rows(x, self.c[0], self.s[0], rows=self.write[:, 0], count=self.starts[0][-1:])
        o.frame_map(lengths, first, self.table, self.ring, self.read[0], self.starts[1], (-1, 0), low=zero, high=last)
        o.linear_int8(self.c[0], self.w1, self.s1, scale=self.s[0], rows=self.read[0], count=self.starts[1][-1:], out=self.low)
        o.quantize_rows(self.low, self.c[1], self.s[1], rows=self.write[:, 0], count=self.starts[0][-1:])
        o.frame_map(lengths, first, self.table, self.ring, self.read[1], self.starts[2], (-2, 0), low=zero, high=last)
        o.linear_int8(self.c[1], self.w2, self.s2, scale=self.s[1], rows=self.read[1], count=self.starts[2][-1:], bias=self.bias,
                      relu=True, gain=self.gain, shift=self.shift, residual=x, residual_scale=0.75, out=self.out)
        return self.out


def _layer_reference(L, xs, lens):
    """The layer over every stream's whole history in 64 bits, frame by frame; the frames of the last step."""
    h = [[] for _ in range(L.streams)]
    for x, lengths in zip(xs, lens):
        at = 0
        for r, n in enumerate(lengths):
            h[r] += list(x[at:at + n])
            at += n
    outs, tol = [], []
    for r in range(L.streams):
        x = np.array(h[r])
        n, t = lens[-1][r], np.arange(len(h[r]))
        c, s = ref.codes_of(x)
        low, _ = ref.linear(c, s, np.stack([np.maximum(t - 1, 0), t], 1), L.w1.cpu().numpy(), L.s1.cpu().numpy(), 2)
        c2, s2 = ref.codes_of(low.astype(np.float32))
        v, size = ref.linear(c2, s2, np.stack([np.maximum(t - 2, 0), t], 1), L.w2.cpu().numpy(), L.s2.cpu().numpy(), 2, bias=_np(L.bias),
                             relu=True, gain=_np(L.gain), shift=_np(L.shift), residual=x, residual_scale=0.75)
        # a bottleneck value within rounding of a half may take the next code: one step of its scale
        # times the largest weight of its column, for each of a few such values
        w2 = np.abs(L.w2.cpu().numpy().astype(np.float64)).max(1) * L.s2.cpu().numpy() * np.abs(_np(L.gain))
        step = np.array([max(s2[max(0, i - 2)], s2[i]) for i in t])[:, None] * w2
        outs.append(v[len(x) - n:])
        tol.append((12 * 2.0 ** -24 * size + 4 * step)[len(x) - n:])
    return np.concatenate(outs), np.concatenate(tol)


def _steps(g, L, n):
    """n steps of ragged streams: (x, lengths) on the GPU, packed."""
    out = []
    for i in range(n):
        lens = [L.frames - (r + i) % 3 for r in range(L.streams)]
        x = _randn(g, L.streams * L.frames, L.dim)
        out.append((x, lens))
    return out


def _limits(L, lens, first):
    dev = dict(dtype=torch.int32, device="cuda")
    lengths, f = torch.tensor(lens, **dev), torch.tensor(first, **dev)
    return lengths, f, torch.zeros(L.streams, **dev), f + lengths - 1


def test_streaming_layers_equal_the_whole_utterance(ops):
    """Step after step through the caches gives what the whole history gives."""
    g = _gen(21)
    L = _Layer(ops, g, 5, 12, 80, 24)
    first, xs, lens = [0] * L.streams, [], []
    for x, ln in _steps(g, L, 8):
        lengths, f, zero, last = _limits(L, ln, first)
        y = L.step(x, lengths, f, zero, last)
        xs.append(_np(x))
        lens.append(ln)
        want, tol = _layer_reference(L, xs, lens)
        got = _np(y)[:len(want)]
        assert (np.abs(got - want) <= tol).all()
        exact = np.abs(got - want) <= 20 * 2.0 ** -24 * (1 + np.abs(want))
        assert exact.mean() > 0.9  # and nearly every row takes no other code
        first = [a + b for a, b in zip(first, ln)]


def test_captured_steps_equal_eager_ones(ops):
    """The run of operators captured once and replayed over new inputs, eager
    work between the replays, against eager calls."""
    g = _gen(22)
    A, B = (_Layer(ops, _gen(23), 4, 9, 64, 20) for _ in range(2))
    steps = _steps(g, A, 7)
    first = [0] * 4
    x = steps[0][0].clone()
    lengths, f, zero, last = (t.clone() for t in _limits(A, steps[0][1], first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        A.step(x, lengths, f, zero, last)  # warm, and writes what the first replay writes again
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.step(x, lengths, f, zero, last)
    for xs, ln in steps:
        now = _limits(A, ln, first)
        x.copy_(xs)
        for to, v in zip((lengths, f, zero, last), now):
            to.copy_(v)
        graph.replay()
        want = B.step(xs, *now)
        torch.cuda.synchronize()
        assert torch.equal(A.out, want)
        for a, b in zip(A.c + A.s, B.c + B.s):
            assert torch.equal(a, b)
        first = [a + b for a, b in zip(first, ln)]


@pytest.mark.parametrize("m", [1, 12, 300])
def test_captured_float_product(ops, m):
    """Float rows quantised in the call: the workspace belongs to the graph; two graphs and eager calls by turns."""
    g = _gen(m)
    w, ws = ops.quantize_weight(_randn(g, 130, 200))
    xs = [_randn(g, m, 200) for _ in range(2)]
    ops.linear_int8(xs[0], w, ws)
    outs, graphs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.linear_int8(x, w, ws))
        graphs.append(graph)
    for i in range(5):
        for x in xs:
            x.copy_(_randn(g, m, 200))
        for gr in graphs:
            gr.replay()
        want = [ops.linear_int8(x, w, ws) for x in xs]
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_two_streams_at_once(ops):
    """The same operators on two streams at once, each with its own outputs."""
    g = _gen(31)
    w, ws = ops.quantize_weight(_randn(g, 300, 256))
    xs = [_randn(g, 500, 256) for _ in range(2)]
    want = [ops.linear_int8(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.linear_int8(xs[i], w, ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_results_do_not_change_from_call_to_call(ops):
    g = _gen(41)
    w, ws = ops.quantize_weight(_randn(g, 777, 1000))
    for m in (1, 9, 40, 1999):
        x = _randn(g, m, 1000)
        first = ops.linear_int8(x, w, ws, dtype=torch.bfloat16)
        for _ in range(3):
            assert torch.equal(ops.linear_int8(x, w, ws, dtype=torch.bfloat16), first)


def test_a_row_does_not_depend_on_the_rows_beside_it(ops):
    """A stream's outputs are the same bits alone and in a batch."""
    g = _gen(42)
    for n, k, taps in ((512, 96, 2), (96, 512, 2), (2000, 192, 1)):
        c, s = ops.quantize_rows(_randn(g, 400, k))
        w, ws = ops.quantize_weight(_randn(g, n, taps * k), taps)
        rows = torch.randint(0, 400, (700, taps), generator=g, device="cuda", dtype=torch.int32)
        y = ops.linear_int8(c, w, ws, scale=s, rows=rows)
        for a, b in ((0, 1), (5, 22), (100, 133), (300, 420)):
            assert torch.equal(ops.linear_int8(c, w, ws, scale=s, rows=rows[a:b].contiguous()), y[a:b])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_another_device_than_the_current_one(ops):
    with torch.cuda.device(1):
        x = torch.randn(5, 100, device="cuda:1")
        w, ws = ops.quantize_weight(torch.randn(9, 100, device="cuda:1"))
        want = ops.linear_int8(x, w, ws)
    with torch.cuda.device(0):
        assert torch.equal(ops.linear_int8(x, w, ws), want)


# ---- largest launches


def test_quantize_rows_of_more_rows_than_a_dimension_of_the_grid(ops):
    m = (1 << 26) + 5  # a launch has less than 2^32 threads a dimension: 64 threads a row here
    x = (torch.arange(m, device="cuda", dtype=torch.int32) % 251 - 125).float()[:, None]
    codes = torch.full((m, 64), 3, dtype=torch.int8, device="cuda")
    scales = torch.full((m,), -1.0, device="cuda")
    ops.quantize_rows(x, codes, scales)
    want = x[:251].abs().cpu()[:, 0].numpy() / np.float32(127)
    assert torch.equal(scales, torch.from_numpy(want).cuda()[torch.arange(m, device="cuda") % 251])
    assert torch.equal(codes[:, 0].float(), 127 * torch.sign(x[:, 0]))
    assert not codes[:, 1:].any()


def test_linear_of_more_rows_than_a_dimension_of_the_grid(ops):
    m, c, g = 1 << 30, 1009, _gen(81)  # 2^24 tiles of 64 rows by 256 threads: 2^32
    codes, scales = ops.quantize_rows(_randn(g, c, 40))
    w, ws = ops.quantize_weight(_randn(g, 1, 40))
    few = ops.linear_int8(codes, w, ws, scale=scales, dtype=torch.float16)
    rows = torch.arange(c, device="cuda", dtype=torch.int32).repeat(-(-m // c))[:m, None]
    out = torch.full((m, 1), 7.0, dtype=torch.float16, device="cuda")
    ops.linear_int8(codes, w, ws, scale=scales, rows=rows, out=out)
    whole = m // c * c
    assert (out[:whole].view(-1, c) == few.view(1, c)).all()
    assert torch.equal(out[whole:], few[:m - whole])


def test_frame_map_rows_past_31_bits_have_no_entry(ops):
    """Pages so high that a cache row's number passes 2^31 - 1."""
    page = 1 << 20
    table = torch.tensor([[2047, 2048, 2047, 1 << 30], [2**31 - 1, 0, 1, 4096]], dtype=torch.int32, device="cuda")
    first = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    rows = torch.full((8, 2), 9, dtype=torch.int32, device="cuda")
    ops.frame_map(lengths, first, table, page, rows, offsets=(0, 1), step=1)
    assert rows[:4].tolist() == [[2047 * page + i, 2047 * page + i + 1] for i in range(4)]
    assert (rows[4:] == -1).all()
    for q, want in ((1, -1), (2, 2047 * page), (3, -1)):
        ops.frame_map(lengths[:1], torch.tensor([q * page], dtype=torch.int32, device="cuda"), table[:1], page, rows[:4],
                      offsets=(0, page - 1))
        assert rows[:4, 0].tolist() == [want + i if want >= 0 else -1 for i in range(4)]
    # page * frame_stride past 32 bits as well
    ops.frame_map(lengths[:1], first[:1], table[:1], page, rows[:4], offsets=(5, page - 4), strides=(1, 4096))
    assert rows[:4, 0].tolist() == [2047 + (5 + i) * 4096 for i in range(4)]
    assert (rows[:4, 1] == -1).all()


def test_captured_map_of_many_streams(ops):
    """More streams than a workgroup sums by itself (two launches), replayed with other lengths."""
    g, r = _gen(82), 5000
    lengths = torch.randint(0, 9, (r,), generator=g, device="cuda", dtype=torch.int32)
    first = torch.randint(0, 4000, (r,), generator=g, device="cuda", dtype=torch.int32)
    table = torch.randint(0, 99999, (r, 3), generator=g, device="cuda", dtype=torch.int32)
    rows = torch.full((9 * r, 2), -7, dtype=torch.int32, device="cuda")
    starts = torch.empty(r + 1, dtype=torch.int32, device="cuda")
    ops.frame_map(lengths, first, table, 32, rows, starts=starts, offsets=(-3, 0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.frame_map(lengths, first, table, 32, rows, starts=starts, offsets=(-3, 0))
    for i in range(4):
        lengths.copy_(torch.randint(0, 9, (r,), generator=g, device="cuda", dtype=torch.int32))
        rows.fill_(-7)
        graph.replay()
        want = torch.full_like(rows, -7)
        want_starts, _ = ops.frame_map(lengths, first, table, 32, want, offsets=(-3, 0))
        assert torch.equal(starts, want_starts) and torch.equal(rows, want), i


def test_numbers_that_do_not_fit_are_refused(ops):
    g = _gen(83)
    codes, scales = ops.quantize_rows(_randn(g, 3, 64))
    w, ws = ops.quantize_weight(_randn(g, 5, 64))
    for bad in ("1", 1e39, None):
        with pytest.raises(ValueError, match="residual_scale"):
            ops.linear_int8(codes, w, ws, scale=scales, residual_scale=bad)
    with pytest.raises(ValueError, match="gradient"):
        ops.linear_int8(codes, w, ws.clone().requires_grad_(), scale=scales)


@pytest.mark.parametrize("m,k,t", [(1030, 1000, "fp32"), (2051, 2041, "fp32"), (4099, 2041, "bf16"), (4099, 1500, "fp16")])
def test_quantize_rows_of_many_long_rows(ops, m, k, t):
    """So many that a wave takes a row of its own."""
    g = _gen(84)
    x = (_randn(g, m, k) * torch.exp(_randn(g, m, 1))).to(TYPES[t])
    codes, scales = ops.quantize_rows(x)
    _same_codes(codes, scales, x)
    few, few_s = ops.quantize_rows(x[:5].contiguous())
    assert torch.equal(codes[:5], few) and torch.equal(scales[:5], few_s)


@pytest.mark.parametrize("m,n,k,taps", [(40, 300, 576, 1), (64, 4096, 64, 1), (200, 600, 192, 3), (257, 520, 448, 2), (15, 33, 64, 16),
                                        (500, 512, 640, 1), (2049, 520, 1088, 1), (2049, 130, 320, 5), (1999, 300, 832, 2)])
def test_linear_tiles_of_every_size_agree(ops, m, n, k, taps):
    """A row's result is the same in whichever tile it lies: all rows at once, and its own few."""
    g = _gen(m + n)
    codes, scales = ops.quantize_rows(_randn(g, m, k))
    w, ws = ops.quantize_weight(_randn(g, n, taps * k), taps)
    rows = torch.randint(-1, m, (m, taps), generator=g, device="cuda", dtype=torch.int32)
    b, r = _randn(g, n), _randn(g, m, n)
    kw = dict(scale=scales, bias=b, relu=True, gain=b, shift=b, residual_scale=0.7)
    whole = ops.linear_int8(codes, w, ws, rows=rows, residual=r, **kw)
    for lo, hi in ((0, 1), (m // 3, m // 3 + 12), (m - 17, m), (m // 2, min(m, m // 2 + 40))):
        lo = max(lo, 0)
        assert torch.equal(whole[lo:hi], ops.linear_int8(codes, w, ws, rows=rows[lo:hi], residual=r[lo:hi], **kw)), (lo, hi)
    _linear_case(ops, m, n, k, taps, "bf16", "fp32", "brgs", m + n, cache=m)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", [(1, 16384), (1, 16385), (2, 8192), (3, 5440), (16, 1024), (17, 960), (32, 512), (31, 528)])
def test_linear_float_rows_at_the_end_of_one_launch(ops, m, k, t):
    """16384 values (rows x padded columns) are quantised in the product's launch, more before it."""
    _linear_case(ops, m, 45, k, 1, t, "fp32", "brg", m + k)


@pytest.mark.parametrize("count", [0, 1, 5, 19, 50])
@pytest.mark.parametrize("k", [30, 600])
def test_linear_float_rows_through_a_map_up_to_a_count(ops, k, count):
    g, m, n = _gen(85), 20, 70
    x = _randn(g, 33, k).bfloat16()
    w, ws = ops.quantize_weight(_randn(g, n, 2 * k), 2)
    rows = torch.randint(-1, 33, (m, 2), generator=g, device="cuda", dtype=torch.int32)
    cnt = torch.tensor([count], dtype=torch.int32, device="cuda")
    out = torch.full((m, n), 7.0, device="cuda")
    ops.linear_int8(x, w, ws, rows=rows, count=cnt, out=out)
    codes, scales = ops.quantize_rows(x)
    want = ops.linear_int8(codes, w, ws, scale=scales, rows=rows)
    assert torch.equal(out[:count], want[:count]) and (out[count:] == 7.0).all()


@pytest.mark.parametrize("m,n,k,taps", [(4, 30, 64, 1), (40, 300, 320, 2), (70, 600, 512, 1), (300, 1100, 128, 3), (2100, 2000, 256, 2),
                                        (4200, 2200, 320, 1)])
def test_linear_absent_rows_add_nothing_to_anything(ops, m, n, k, taps):
    """The row that stands in for absent ones holds a NaN, and so does every row that no entry names."""
    g = _gen(86)
    x = _randn(g, 64, k)
    x[0, 3], x[1, 0], x[63, k - 1] = float("nan"), float("inf"), float("nan")
    codes, scales = ops.quantize_rows(x)
    w, ws = ops.quantize_weight(_randn(g, n, taps * k), taps)
    b = _randn(g, n)
    rows = torch.randint(2, 63, (m, taps), generator=g, device="cuda", dtype=torch.int32)
    rows[::2, 0] = -1
    rows[1::4, taps - 1] = 64
    rows[m - 1] = 2**31 - 1
    y = ops.linear_int8(codes, w, ws, scale=scales, rows=rows, bias=b)
    assert torch.isfinite(y).all() and torch.equal(y[m - 1], b)
    if taps == 1:
        assert torch.equal(y[::2], b.expand(len(y[::2]), n))
    rows[m // 2, taps - 1] = 63
    bad = ops.linear_int8(codes, w, ws, scale=scales, rows=rows, bias=b)
    assert bad[m // 2].isnan().all()
    bad[m // 2] = y[m // 2]
    assert torch.equal(bad, y)
    rows[m // 2, taps - 1] = -1
    assert torch.equal(ops.linear_int8(x, w, ws, rows=rows, bias=b), ops.linear_int8(codes, w, ws, scale=scales, rows=rows, bias=b))


def test_products_on_two_threads(ops):
    """The C calls of two threads, each on a stream of its own."""
    import threading
    g = _gen(87)
    jobs = []
    for m, n, k in ((5, 200, 300), (90, 500, 640), (600, 700, 512)):
        x = _randn(g, m, k)
        w, ws = ops.quantize_weight(_randn(g, n, k))
        jobs.append((x, w, ws, ops.linear_int8(x, w, ws)))
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(40):
                for x, w, ws, want in jobs:
                    if not torch.equal(ops.linear_int8(x, w, ws), want):
                        bad.append(tuple(x.shape))
        s.synchronize()
    ts = [threading.Thread(target=work) for _ in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k,taps", [(1, 17, 64, 1), (9, 33, 128, 2), (70, 96, 192, 1), (300, 513, 192, 2), (3000, 2000, 96, 1)])
def test_linear_in_place_through_one_map(ops, m, n, k, taps, t):
    """out is the residual and both have the same map; and out is other columns of the residual's rows."""
    g = _gen(m + n + k)
    c, s = ops.quantize_rows(_randn(g, 40, k))
    w, ws = ops.quantize_weight(_randn(g, n, taps * k) / (taps * k) ** 0.5, taps)
    at = torch.randint(-1, 41, (m, taps), generator=g, device="cuda", dtype=torch.int32)
    to = (torch.randperm(m + 30, generator=g, device="cuda")[:m].int() - 10).contiguous()
    a, b = at.cpu().numpy(), to.cpu().numpy()
    ok = (b >= 0) & (b < m + 5)
    big = _randn(g, m + 5, 2 * n + 3).to(TYPES[t])
    res = big[:, :n]
    before = _np(big)
    v, size = ref.linear(c.cpu().numpy(), s.cpu().numpy(), a, w.cpu().numpy(), ws.cpu().numpy(), taps,
                         residual=np.where(ok[:, None], before[np.where(ok, b, 0), :n], 0.0), residual_scale=-1.5)
    for lo in (0, n + 1):  # in place, and beside it
        into = big.clone()
        out = into[:, lo:lo + n]
        ops.linear_int8(c, w, ws, scale=s, rows=at, residual=into[:, :n], residual_scale=-1.5, out=out, out_rows=to, residual_rows=to)
        got = _np(into)
        _check(torch.from_numpy(got[b[ok], lo:lo + n]), v[ok], size[ok], taps, t)
        got[b[ok], lo:lo + n] = before[b[ok], lo:lo + n]
        np.testing.assert_array_equal(got, before)


def test_linear_out_over_the_residual_otherwise_is_refused(ops):
    g = _gen(1)
    x = _randn(g, 50, 64)
    w, ws = ops.quantize_weight(_randn(g, 32, 64))
    buf = _randn(g, 51, 70)
    before = buf.clone()
    to = torch.arange(50, device="cuda", dtype=torch.int32).flip(0).contiguous()
    for kw in (dict(out=buf[:50, :32], residual=buf[:50, :32], out_rows=to), dict(out=buf[:50, :32], residual=buf[:50, :32], residual_rows=to),
               dict(out=buf[:50, :32], residual=buf[:50, :32], out_rows=to, residual_rows=to.clone()),
               dict(out=buf[:50, :32], residual=buf[:50, 31:63]), dict(out=buf[:50, :32], residual=buf[1:, :32]),
               dict(out=buf[:50, :32], residual=buf[1:, :32], out_rows=to, residual_rows=to)):
        with pytest.raises(ValueError, match="overlap"):
            ops.linear_int8(x, w, ws, **kw)
    assert torch.equal(buf, before)


@pytest.mark.parametrize("floats", [False, True])
@pytest.mark.parametrize("m", [3, 20, 300])
def test_linear_residual_of_no_rows_adds_nothing(ops, m, floats):
    """res_rows = 0: no row is read, whatever the map names and wherever the matrix lies."""
    g = _gen(m)
    x = _randn(g, m, 64)
    w, ws = ops.quantize_weight(_randn(g, 40, 64))
    codes, scales = ops.quantize_rows(x)
    kw = dict(scale=None if floats else scales)
    want = ops.linear_int8(x if floats else codes, w, ws, **kw)
    rows = torch.randint(-2, 5, (m,), generator=g, device="cuda", dtype=torch.int32)
    got = ops.linear_int8(x if floats else codes, w, ws, residual=torch.zeros(0, 40, device="cuda"), residual_rows=rows, **kw)
    assert torch.equal(got, want)
    # the same in C, with an address: that of a matrix of NaN
    nan = torch.full((8, 40), float("nan"), device="cuda")
    out, space = torch.zeros_like(want), torch.empty(m * 68, dtype=torch.int8, device="cuda")
    p = [t.data_ptr() for t in (codes, scales, x, space, w, ws, nan, out, rows)]
    args = ops._LINEAR(*(0, 0, 0, 0, p[2], p[3]) if floats else (p[0], p[1], 0, 0, 0, 0), p[4], p[5], 0, 0, 0, p[6], p[7], 0, p[8],
                       m, 0 if floats else 64, 64 if floats else 0, 64, 40, 40, 0, 0, 0, 1, 0, m, 40, 64, 1, 0, 0, 0, 0, 2.0)
    assert ops._c.vamd_op_linear_int8(0, torch.cuda.current_stream().cuda_stream, args) == 0
    assert torch.equal(out, want)


def test_forward_mode_tangents_are_refused(ops):
    import torch.autograd.forward_ad as fw
    g = _gen(2)
    x = _randn(g, 5, 64)
    w, ws = ops.quantize_weight(_randn(g, 8, 64))
    codes, scales = ops.quantize_rows(x)
    y = _randn(g, 5, 8)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.quantize_rows(dual(x)), lambda: ops.quantize_rows(x, codes, dual(scales)), lambda: ops.quantize_weight(dual(x)),
                     lambda: ops.linear_int8(dual(x), w, ws), lambda: ops.linear_int8(x, w, dual(ws)), lambda: ops.linear_int8(codes, w, ws, scale=dual(scales)),
                     lambda: ops.linear_int8(x, w, ws, bias=dual(ws)), lambda: ops.linear_int8(x, w, ws, gain=ws, shift=dual(ws)),
                     lambda: ops.linear_int8(x, w, ws, residual=dual(y)), lambda: ops.linear_int8(x, w, ws, out=dual(y))):
            with pytest.raises(ValueError, match="gradient"):
                call()
        ops.linear_int8(x, w, ws)
    with pytest.raises(ValueError, match="gradient"):
        ops.quantize_rows(x, codes, scales.clone().requires_grad_())
    with pytest.raises((ValueError, RuntimeError)):  # (its tensors have no address)
        torch.func.jvp(lambda a: ops.linear_int8(a, w, ws), (x,), (x,))


def test_a_device_that_is_not_there_leaves_no_error_behind(ops):
    """The call fails and says why; the next launch of the process, whoever's, does not report it again."""
    x = _randn(_gen(0), 4, 64)
    c, s = torch.empty(4, 64, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    torch.cuda.synchronize()
    args = ops._ROWS(x.data_ptr(), 0, 0, 0, c.data_ptr(), s.data_ptr(), 4, 64, 4, 64, 0, 0, 4, 0, 64)
    for device in (torch.cuda.device_count(), -1):
        assert ops._c.vamd_op_quantize_rows(device, None, args) < 0
        assert b"HIP error" in ops._c.vamd_last_error()
        torch.add(x, 1.0)
        ops.quantize_rows(x)
    torch.cuda.synchronize()
