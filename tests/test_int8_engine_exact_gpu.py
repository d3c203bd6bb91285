"""The engine's 8-bit acoustic model bit for bit: every layer of the network
evaluated here in the arithmetic that the engine states for it -- exact
integer sums and 32-bit steps in their order for the 8-bit products, the
canonical 32-bit order for the others -- and the log-likelihoods compared for
equality."""
import numpy as np
import pytest

import int8_ref as ref
import np_kaldi as nk
import oracle_py
from test_int8_engine_gpu import _products, _run

f32 = np.float32


def fma(x, y, z):
    """x * y + z of 32-bit floats, rounded once: the product is exact in 64 bits, the sum is rounded to odd there
    (to the neighbour whose last bit is set, where it is inexact), which leaves the rounding to 32 bits as it would be
    of the sum itself."""
    p, z = np.float64(x) * np.float64(y), np.float64(z)
    s = np.atleast_1d(p + z)
    b = s - p
    e = (p - (s - b)) + (z - b)  # what the sum lost, exactly
    even = (s.view(np.int64) & 1) == 0
    return np.where((e != 0) & even, np.nextafter(s, np.copysign(np.inf, e)), s).astype(f32)


def affine(w, x):
    """W x in the canonical order: K in slices, each a chain of fmas over its k (0, 4, 1, 5, 2, 6, 3, 7 of every eight)."""
    k = w.shape[1]
    n = 1
    if k >= 512 and k % 256 == 0:
        while n < 8 and 2 * n <= k // 256:
            n *= 2
    total = None
    for z in range(n):
        part, end = np.zeros(len(w), f32), (z + 1) * (k // n)
        for g in range(z * (k // n), end, 8):
            for i in (0, 4, 1, 5, 2, 6, 3, 7) if g + 8 <= end else range(end - g):
                part = fma(x[g + i], w[:, g + i], part)
        total = part if total is None else total + part
    return total


class Network(nk.NnetGraph):
    def __init__(self, nn, products):
        super().__init__(nn)
        self.products, self.weights = products, {}

    def product(self, name, w, parts):
        if name not in self.weights:
            c, s = ref.codes_of(w)
            self.weights[name] = c[:, :w.shape[1]].astype(np.float64), s
        wc, ws = self.weights[name]
        v, col = np.zeros(len(w), f32), 0
        for x in parts:
            c, s = ref.codes_of(x[None])
            v = fma((wc[:, col:col + len(x)] @ c[0, :len(x)].astype(np.float64)).astype(f32), s[0], v)
            col += len(x)
        return v * ws

    def component(self, name, parts):
        kind, f = self.nn.components[self.nodes[name]["component"]]
        f = dict(f) if isinstance(f, list) else f
        w = f.get("<LinearParams>", f.get("<Params>"))
        if w is not None:
            w = np.asarray(w, f32)
            y = self.product(name, w, parts) if name in self.products else affine(w, np.concatenate(parts))
            b = f.get("<BiasParams>")
            return y + np.asarray(b, f32) if b is not None and len(b) else y
        assert name not in self.products and len(parts) == 1
        x = parts[0]
        if kind == "RectifiedLinearComponent":
            return np.where(x < 0, f32(0), x)
        if kind == "BatchNormComponent":
            s, o = oracle_py.bn_scale_offset_f32(f)
            return x * np.tile(s, len(x) // len(s)) + np.tile(o, len(x) // len(s))
        assert kind in oracle_py.OracleNet.IDENT, kind
        return x

    def forward(self, feats, ivector_at, times):
        cache = {}

        def node(name, t):
            if (name, t) not in cache:
                nd = self.nodes[name]
                if nd["kind"] == "input":
                    v = feats[min(max(t, 0), len(feats) - 1)]
                elif nd["kind"] == "dimrange":
                    v = node(nd["src"], t)[nd["offset"]:nd["offset"] + nd["dim"]]
                elif nd["kind"] == "output":
                    v = desc(nd["input"], t)
                else:
                    kind, f = self.nn.components[nd["component"]]
                    offsets = dict(f)["<TimeOffsets>"] if kind == "TdnnComponent" else [0]
                    v = self.component(name, [desc(nd["input"], t + int(o)) for o in offsets])
                assert v.dtype == f32, name
                cache[name, t] = v
            return cache[name, t]

        def desc(d, t):
            k = d[0]
            if k == "node":
                return node(d[1], t)
            if k == "offset":
                return desc(d[1], t + d[2])
            if k == "scale":
                return f32(d[1]) * desc(d[2], t)
            if k == "sum":
                y = desc(d[1][0], t)
                for e in d[1][1:]:
                    y = y + desc(e, t)
                return y
            if k == "append":
                return np.concatenate([desc(e, t) for e in d[1]])
            if k == "ifdefined":
                return desc(d[1], t)
            if k == "const":
                return np.full(d[2], d[1], f32)
            assert k == "replace_index" and d[1] == ("node", "ivector"), k
            return ivector_at(t)

        return np.stack([node("output", t) for t in times])


def log_likelihoods(model, wave, products, frames):
    """The last `frames` output frames of the wave and the first."""
    o = oracle_py.OracleModel(model, fpc=51)
    raw = o.features(wave)
    iv = o.ivectors(raw) if o.ivector is not None else None
    of, t0 = o._ivec_of_time(len(raw), len(iv)) if iv is not None else (None, 0)
    times = range(0, len(raw), o.fss)
    rows = sorted({*range(min(frames, len(times))), *range(max(0, len(times) - frames), len(times))})
    y = Network(o.nn, products).forward(np.asarray(o.nnet_features(raw), f32), lambda t: iv[of[t - t0]],
                                        [times[r] for r in rows])
    return rows, y * f32(o.acoustic_scale)


def test_the_evaluation_itself(synth_model, test_wave):
    """Without products it is the 32-bit oracle's, bit for bit; fma against exact fractions."""
    from fractions import Fraction
    rng = np.random.default_rng(3)
    x, y, z = (rng.standard_normal(300).astype(f32) * f32(2.0) ** rng.integers(-40, 40, 300).astype(f32) for _ in range(3))
    z[:100] = -(x[:100] * y[:100])  # all but the product's last bits cancel
    z[100:200] = (x[100:200] * y[100:200]) * f32(2.0 ** 25)
    for a, b, c, got in zip(x, y, z, fma(x, y, z)):
        want = Fraction(float(a)) * Fraction(float(b)) + Fraction(float(c))
        near = [np.nextafter(got, f32(-np.inf)), got, np.nextafter(got, f32(np.inf))]
        off = [abs(Fraction(float(v)) - want) for v in near]
        assert off[1] <= min(off[0], off[2]) and (off[1] < min(off[0], off[2]) or got.view(np.int32) % 2 == 0), (a, b, c)
    wave = test_wave[:16000]
    rows, y = log_likelihoods(synth_model, wave, set(), 2)
    np.testing.assert_array_equal(y, oracle_py.OracleModel(synth_model, fpc=51).loglikes(wave)[rows])


@pytest.mark.gpu
def test_log_likelihoods_equal_the_stated_arithmetic(synth_model, test_wave):
    wave = test_wave[:16000 * 2]
    e, _, (llh,) = _run(synth_model, [wave])
    products = _products(synth_model)
    assert e.int8_layers == len(products) == 24
    rows, y = log_likelihoods(synth_model, wave, products, 12)
    np.testing.assert_array_equal(llh[rows], y)


@pytest.mark.gpu
def test_many_streams_equal_the_stated_arithmetic(synth_model, test_wave):
    """The tiled products: 90 streams of one wave, and two others among them."""
    waves = [test_wave[:16000]] * 92
    waves[7], waves[91] = test_wave[20000:36000], test_wave[40000:52345]
    _, _, llh = _run(synth_model, waves)
    products = _products(synth_model)
    for i in (7, 90, 91):
        rows, y = log_likelihoods(synth_model, waves[i], products, 4)
        np.testing.assert_array_equal(llh[i][rows], y, err_msg=str(i))


@pytest.mark.gpu
def test_other_front_ends_equal_the_stated_arithmetic(synth_model_frontend, test_wave):
    wave = test_wave[:16000]
    _, _, (llh,) = _run(synth_model_frontend, [wave])
    rows, y = log_likelihoods(synth_model_frontend, wave, _products(synth_model_frontend), 4)
    np.testing.assert_array_equal(llh[rows], y)
