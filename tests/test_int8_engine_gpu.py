"""The engine's 8-bit acoustic model (Engine(precision="int8"), VOSK_AMD_NNET):
the layers' wiring against a plain evaluation of the same network with
quantised layers, and that nothing of a stream's result depends on what runs
beside it."""
import json
import os

import numpy as np
import pytest

import int8_ref as ref
import np_kaldi as nk
import oracle_py
from conftest import perturbed_stream

pytestmark = pytest.mark.gpu


def _run(model, waves, precision="int8", pipeline=False, fpc=51, chunk=None):
    """Log-likelihoods of every stream, all fed together."""
    from vosk import engine
    e = engine.Engine(model, frames_per_chunk=fpc, max_streams=len(waves), keep_llh=True, pipeline=pipeline, precision=precision)
    ss = [e.new_stream() for _ in waves]
    if pipeline:
        for s, w in zip(ss, waves):
            e.preload(s, w, finished=True)
        while e.step(ss):
            pass
        e.flush()
    elif chunk:
        for i in range(0, max(len(w) for w in waves), chunk):
            for s, w in zip(ss, waves):
                if i < len(w):
                    e.accept(s, w[i:i + chunk])
            e.advance(ss)
        for s in ss:
            e.accept(s, np.zeros(0, np.float32), finished=True)
        e.advance(ss)
    else:
        for s, w in zip(ss, waves):
            e.accept(s, w, finished=True)
        e.advance(ss)
    return e, ss, [e.llh(s) for s in ss]


class _Quantised(nk.NnetGraph):
    """The network in 64 bits with the products' inputs and weights in codes
    and the layers' outputs rounded to 32-bit floats, as their rings hold them."""

    def __init__(self, nn, products):
        super().__init__(nn)
        self.products, self.weights = products, {}

    def quantised(self, name, f, parts):
        w = f["<LinearParams>"] if "<LinearParams>" in f else f["<Params>"]
        if name not in self.weights:
            c, s = ref.codes_of(w)
            self.weights[name] = c[:, :w.shape[1]].astype(np.float64), s.astype(np.float64)
        wc, ws = self.weights[name]
        y, col = 0.0, 0
        for x in parts:
            c, s = ref.codes_of(x.astype(np.float32)[None])
            y = y + float(s[0]) * (wc[:, col:col + len(x)] @ c[0, :len(x)])
            col += len(x)
        y = y * ws
        b = f.get("<BiasParams>")
        return y + b if b is not None and len(b) else y

    def forward(self, inputs, t_out):
        cache, comps = {}, self.nn.components

        def node(name, t):
            key = (name, t)
            if key not in cache:
                nd = self.nodes[name]
                if nd["kind"] == "input":
                    cache[key] = inputs[name][min(max(t, 0), len(inputs[name]) - 1)]
                elif nd["kind"] == "output":
                    cache[key] = desc(nd["input"], t)
                else:
                    kind, f = comps[nd["component"]]
                    f = dict(f) if isinstance(f, list) else f
                    offs = f["<TimeOffsets>"] if kind == "TdnnComponent" else [0]
                    parts = [desc(nd["input"], t + o) for o in offs]
                    if name in self.products:
                        v = self.quantised(name, f, parts)
                    else:
                        v = nk.apply_component(kind, f, np.concatenate(parts))
                    cache[key] = v
            return cache[key]

        def desc(d, t):
            k = d[0]
            if k == "node":
                return node(d[1], t)
            if k == "offset":
                return desc(d[1], t + d[2])
            if k == "scale":
                return d[1] * desc(d[2], t)
            if k == "sum":
                return sum(desc(e, t) for e in d[1])
            if k == "append":
                return np.concatenate([desc(e, t) for e in d[1]])
            assert k == "replace_index"
            return inputs["ivector_at"](t)

        return np.stack([node("output", t) for t in t_out])


def _products(model):
    from vosk import engine
    ops = [ln.split(":")[0] for ln in engine.plan_describe_int8(model, 51).splitlines()[:-1] if "product of" in ln]
    names = {"prefinal-chain.batchnorm1": "prefinal-chain.affine", "prefinal-chain.batchnorm2": "prefinal-chain.linear",
             "tdnn1.dropout": "tdnn1.affine"}
    return {names.get(o, o.replace(".noop", ".affine")) for o in ops}


def _rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


def test_layers_against_a_plain_quantised_network(synth_model, test_wave):
    """Rounding an activation to 1 of 255 codes errs by a step / sqrt(12), 1.3 %
    of its rms where the largest of a few hundred is 5.6 times the rms; a
    weight by 0.8 %.  24 layers of it add up to about 7.5 % in quadrature.  The
    two evaluations round the same way but where 32-bit arithmetic put a value
    on the other side of a half, after which the codes of later layers may
    differ as two independent roundings do at the most: sqrt(2) * 1.3 % a
    layer, 9 % in all.  A wrong tap, scale, bypass or column errs by the size of
    the values themselves."""
    wave = test_wave[:16000 * 2]
    e, (s,), (llh,) = _run(synth_model, [wave])
    assert e.int8_layers == 24
    fp32 = _run(synth_model, [wave], "fp32")
    assert fp32[0].int8_layers == 0
    spread = _rms(llh - llh.mean(0))
    off = _rms(llh - fp32[2][0])
    assert 0 < off < 0.2 * spread, (off, spread)

    o = oracle_py.OracleModel(synth_model, fpc=51)
    raw = o.features(wave)
    np.testing.assert_array_equal(e.ivectors(s), o.ivectors(raw))  # the front end is the same
    iv = o.ivectors(raw)
    of, t0 = o._ivec_of_time(len(raw), len(iv))
    g = _Quantised(o.nn, _products(synth_model))
    t_out = list(range(0, len(raw), 3))[:20]
    want = g.forward({"input": o.nnet_features(raw).astype(np.float64), "ivector_at": lambda t: iv[of[t - t0]].astype(np.float64)}, t_out)
    got = llh[:20]
    assert _rms(got - want) < 0.09 * spread, (_rms(got - want), spread)
    # and they differ less than either does from 32 bits
    assert _rms(got - want) < _rms(got - fp32[2][0][:20])


def test_a_stream_alone_in_a_batch_and_in_the_pipeline(synth_model, test_wave):
    """The same bits with 1, 3 and 40 streams (few-row and tiled products), chunk sizes, in order and pipelined."""
    waves = [perturbed_stream(test_wave, i, seconds=1.0 + 0.07 * (i % 9)) for i in range(40)]
    _, _, batch = _run(synth_model, waves)
    for i in (0, 7, 39):
        _, _, (alone,) = _run(synth_model, [waves[i]])
        np.testing.assert_array_equal(alone, batch[i])
    _, _, three = _run(synth_model, waves[:3], chunk=3200)
    _, _, piped = _run(synth_model, waves, pipeline=True)
    for i in range(3):
        np.testing.assert_array_equal(three[i], batch[i])
    for a, b in zip(piped, batch):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("fpc", [21, 51, 150])
def test_chunk_sizes_and_reused_streams(synth_model, test_wave, fpc):
    """Another chunk size, and a stream slot that an earlier, longer stream has used."""
    from vosk import engine
    wave = test_wave[:16000]
    e = engine.Engine(synth_model, frames_per_chunk=fpc, max_streams=2, keep_llh=True, precision="int8")
    s = e.new_stream()
    e.accept(s, test_wave[:50000], finished=True)
    e.advance([s])
    e.free_stream(s)
    s = e.new_stream()
    e.accept(s, wave, finished=True)
    e.advance([s])
    _, _, (fresh,) = _run(synth_model, [wave], fpc=fpc)
    np.testing.assert_array_equal(e.llh(s), fresh)
    assert np.isfinite(fresh).all()


def test_environment_and_public_api(synth_model, test_wave, monkeypatch):
    """VOSK_AMD_NNET reaches every engine, the recognizers' and the batch model's among them."""
    import vosk
    from vosk import engine
    monkeypatch.setenv("VOSK_AMD_NNET", "int8")
    e = engine.Engine(synth_model, max_streams=1)
    assert e.int8_layers == 24
    e.close()
    vosk.SetLogLevel(-1)
    m = vosk.Model(synth_model)
    rec = vosk.KaldiRecognizer(m, 16000)
    pcm = np.asarray(test_wave[:48000], np.float32).astype("<i2").tobytes()
    rec.AcceptWaveform(pcm)
    assert "text" in json.loads(rec.FinalResult())
    monkeypatch.setenv("VOSK_AMD_NNET", "fp32")
    e = engine.Engine(synth_model, max_streams=1, precision="int8")
    assert e.int8_layers == 0
    e.close()
    monkeypatch.setenv("VOSK_AMD_NNET", "int9")
    with pytest.raises(RuntimeError, match="VOSK_AMD_NNET"):
        engine.Engine(synth_model, max_streams=1)


def test_other_front_ends(synth_model_frontend, test_wave):
    """Models with another front end (log fbank, CMVN on the input)."""
    e, _, (llh,) = _run(synth_model_frontend, [test_wave[:16000]])
    _, _, (fp,) = _run(synth_model_frontend, [test_wave[:16000]], "fp32")
    assert e.int8_layers == 24
    assert 0 < _rms(llh - fp) < 0.2 * _rms(fp - fp.mean(0))


def test_more_streams_than_threads_of_a_map(synth_model, test_wave):
    """A pass of 260 jobs: the row maps' other form; every stream as it is alone."""
    waves = [perturbed_stream(test_wave, i % 3, seconds=1.0 + 0.2 * (i % 3)) for i in range(260)]
    e, ss, llh = _run(synth_model, waves)
    e.close()
    for i in range(3):
        e, _, alone = _run(synth_model, [waves[i]])
        e.close()
        for k in range(i, 260, 3):
            np.testing.assert_array_equal(llh[k], alone[0], err_msg=str(k))


def _batch_texts(model_dir, waves, monkeypatch):
    import vosk
    monkeypatch.setenv("VOSK_BATCH_MODEL_DIR", model_dir)
    model = vosk.BatchModel()
    recs = [vosk.BatchRecognizer(model, 16000) for _ in waves]
    for r, w in zip(recs, waves):
        r.AcceptWaveform(np.asarray(w, np.float32).astype("<i2").tobytes())
        r.FinishStream()
    model.Wait()
    out = []
    for r in recs:
        text = ""
        while True:
            res = r.Result()
            if not res:
                break
            text += " " + json.loads(res)["text"]
        out.append(text.strip())
    return out


def test_batch_model_at_its_own_number_of_streams(synth_model_noep, test_wave, monkeypatch):
    """600 streams and 2 000 outputs: the log-likelihoods have no ring, so no ring's limit is theirs.  The results are
    those of a batch model with 4 streams."""
    import vosk
    vosk.SetLogLevel(-1)
    vosk.GpuInit()
    monkeypatch.setenv("VOSK_AMD_NNET", "int8")
    monkeypatch.delenv("VOSK_AMD_BATCH_SLOTS", raising=False)
    waves = [perturbed_stream(test_wave, i, seconds=2.0 + 0.45 * i) for i in range(3)]
    many = _batch_texts(synth_model_noep, waves, monkeypatch)
    monkeypatch.setenv("VOSK_AMD_BATCH_SLOTS", "4")
    few = _batch_texts(synth_model_noep, waves, monkeypatch)
    assert many == few and all(many), (many, few)


def test_streams_past_the_limit_of_a_ring_are_refused_with_the_number(synth_model):
    """A ring of 512 frames of 512 floats a stream is 1 MiB: 2 047 streams stay below 2^31 bytes."""
    from vosk import engine
    with pytest.raises(RuntimeError, match="at most 2047 streams an engine"):
        engine.Engine(synth_model, frames_per_chunk=51, max_streams=2048, precision="int8")


def test_an_empty_environment_variable_is_none(synth_model, monkeypatch):
    from vosk import engine
    monkeypatch.setenv("VOSK_AMD_NNET", "")
    for precision, layers in (("fp32", 0), ("int8", 24)):
        e = engine.Engine(synth_model, max_streams=1, precision=precision)
        assert e.int8_layers == layers
        e.close()
