"""Engine.score_tokens against the oracle: log probabilities of prompts' own
tokens, entropy and alternatives from its full-vocabulary logits.  The hidden
states differ as in the other parity tests (F16 operands), so log
probabilities are held to the gate of those, 3e-2 at most and 3e-3 on average
on the tiny models; what follows from the GPU's own numbers is exact: repeats,
order of the alternatives."""
import numpy as np
import pytest

import oracle
from laya_goish_b200 import engine, synth
from laya_goish_b200._lib import E_INVALID, LayaError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(tiny_paths):
    out = {n: (engine.Engine(tiny_paths[n]), oracle.Model(open(tiny_paths[n], "rb").read(), threads=8))
           for n in ("tiny-llama-f16", "tiny-llama-q8_0", "tiny-qwen2-f16")}
    yield out
    for e, o in out.values():
        e.close()
        o.close()


def log_softmax(x):
    d = x - x.max(-1, keepdims=True)
    return d - np.log(np.exp(d).sum(-1, keepdims=True))


@pytest.mark.parametrize("name", ["tiny-llama-f16", "tiny-llama-q8_0", "tiny-qwen2-f16"])
def test_score_matches_oracle(models, name):
    e, o = models[name]
    rng = np.random.default_rng(5)
    prompts = [synth.token_ids(rng, o.vocab, n) for n in (2, 70, 1, 33, 129)]
    got = e.score_tokens(prompts, top=4)
    assert [len(g["logprobs"]) for g in got] == [1, 69, 0, 32, 128]
    for ids, g in zip(prompts, got):
        if len(ids) < 2:
            continue
        lp = log_softmax(np.asarray(o.head(o.forward(ids, list(range(len(ids) - 1)))), np.float64))
        want = lp[np.arange(len(ids) - 1), ids[1:]]
        err = np.abs(g["logprobs"] - want)
        assert err.max() < 3e-2 and err.mean() < 3e-3, (err.max(), err.mean())
        ent = -(np.exp(lp) * lp).sum(-1)
        assert np.abs(g["entropy"] - ent).max() < 3e-2
        assert (np.diff(g["top_logprobs"], axis=1) <= 0).all()
        # each alternative is one of the oracle's best, up to the same difference
        own = np.take_along_axis(lp, g["top_ids"].astype(np.int64), 1)
        best = -np.sort(-lp, axis=1)[:, :4]
        assert np.abs(own - g["top_logprobs"]).max() < 3e-2 and np.abs(own - best).max() < 6e-2
    t = e.timing()
    assert t["device_ms"] > 0 and t["launches"] > 0


def test_score_repeats_and_waves(models, monkeypatch):
    e, o = models["tiny-llama-f16"]
    rng = np.random.default_rng(6)
    prompts = [synth.token_ids(rng, o.vocab, n) for n in (40, 130, 7, 65)]
    alone = [e.score_tokens([p], top=3)[0] for p in prompts]
    again = [e.score_tokens([p], top=3)[0] for p in prompts]
    for a, b in zip(alone, again):
        for k in a:
            assert np.array_equal(a[k], b[k]), k
    monkeypatch.setenv("LAYA_WAVE_TOKENS", "100")
    for a, b in zip(alone, e.score_tokens(prompts, top=3)):
        assert np.abs(a["logprobs"] - b["logprobs"]).max() < 1e-2


def test_score_refusals(models):
    e, o = models["tiny-llama-f16"]
    assert e.score_tokens([]) == []
    for prompts, top in (([[]], 0), ([[3, o.vocab]], 0), ([[3, -1]], 0), ([[3, 4]], 65), ([[3, 4]], -1),
                         ([[3] * (e.info["context"] + 1)], 0)):
        with pytest.raises(LayaError) as x:
            e.score_tokens(prompts, top=top)
        assert x.value.code == E_INVALID
    assert e.score_tokens([[3, 4]])[0]["top_ids"].shape == (1, 0)


def test_score_leaves_the_operators_status_word_alone(models):
    """The word in which callers' own operators report (a timeout among them)
    is neither an error of a scoring call nor cleared by it."""
    import ctypes

    from laya_goish_b200 import _lib

    e, o = models["tiny-llama-f16"]
    L = _lib.lib()
    bits = ctypes.c_uint32()
    _lib.check(L.laya_device_status(0, ctypes.byref(bits)))

    class Info(ctypes.Structure):  # of the library's own lookup
        _fields_ = [("device", ctypes.c_int), ("sms", ctypes.c_int), ("status", ctypes.c_uint64)]

    info = Info()
    assert L._ZN4laya11device_infoEPNS_10DeviceInfoE(ctypes.byref(info)) == 0
    pending = ctypes.c_uint32(1 | 2)  # a timeout and a page, as kernels of another caller would leave them
    assert ctypes.CDLL("libcuda.so.1").cuMemcpyHtoD_v2(ctypes.c_uint64(info.status), ctypes.byref(pending),
                                                       ctypes.c_size_t(4)) == 0
    try:
        got = e.score_tokens([[3, 4, 5, 6]], top=2)[0]
    finally:
        _lib.check(L.laya_device_status(0, ctypes.byref(bits)))
    assert np.isfinite(got["logprobs"]).all() and bits.value == 3


def test_score_in_chunks_of_logits():
    """More rows than one chunk of logits holds (256 MB), over an odd vocabulary."""
    path = synth.model_path(synth.Decoder("wide-head-llama-f16", "llama", 1, 256, 4, 2, 512, 40001, 1e4, quant="f16",
                                          seed=18))
    e, o = engine.Engine(path), oracle.Model(open(path, "rb").read(), threads=8)
    rng = np.random.default_rng(8)
    prompts = [synth.token_ids(rng, o.vocab, n) for n in (900, 1, 700, 333)]  # 1930 rows, 1664 to a chunk
    for ids, g in zip(prompts, e.score_tokens(prompts, top=3)):
        if len(ids) < 2:
            continue
        lp = log_softmax(np.asarray(o.head(o.forward(ids, list(range(len(ids) - 1)))), np.float64))
        err = np.abs(g["logprobs"] - lp[np.arange(len(ids) - 1), ids[1:]])
        assert err.max() < 3e-2 and err.mean() < 3e-3, (err.max(), err.mean())
        assert np.abs(g["entropy"] + (np.exp(lp) * lp).sum(-1)).max() < 3e-2
        assert np.abs(np.take_along_axis(lp, g["top_ids"].astype(np.int64), 1) - g["top_logprobs"]).max() < 3e-2
    e.close()
    o.close()
