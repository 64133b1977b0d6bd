"""The Llama engine on the int8 key/value cache (accel_llama_cache): each
layer's cache rows and the logits against a 64-bit form of the same model,
prompts and single tokens, whole and windowed; generation alone and in a
batch; what is refused; and that the fp32 cache's results stay."""

import numpy as np
import pytest

from accelep_b200 import synthetic as syn
from accelep_b200.llama import Llama
from tests import q8_cache_oracle as O

pytestmark = pytest.mark.gpu

CFG = dict(vocab=512, hidden=128, layers=2, heads=2, kv_heads=1, intermediate=256, context=320, eps=1e-5,
           rope_theta=10000.0)
WIDE = dict(CFG, hidden=512, heads=4, kv_heads=2)  # heads of 128


class Model:
    """The model in 64 bits over numpy caches. Attention reads the engine's
    cache rows, so that a value that rounds to the other neighbour in 32 bits
    does not spread; the rows themselves are compared on the way."""

    def __init__(self, cfg, weights, block, window, sinks):
        self.cfg, self.w, self.window, self.sinks = cfg, {k: v.astype(np.float64) for k, v in weights.items()}, window, sinks
        self.d = cfg["hidden"] // cfg["heads"]
        self.tables = O.tables(cfg["context"], self.d, cfg["rope_theta"])
        self.caches = [O.Cache(1, cfg["kv_heads"], cfg["context"], self.d, block) for _ in range(cfg["layers"])]

    def norm(self, x, kind, layer):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg["eps"]) * self.w[(kind, layer)]

    def forward(self, ids, pos0, engine):
        c, w, d = self.cfg, self.w, self.d
        heads, kv, n = c["heads"], c["kv_heads"], len(ids)
        x = w[(syn.W_EMBED, -1)][ids]
        for layer in range(c["layers"]):
            a = self.norm(x, syn.W_ATTN_NORM, layer)
            q, k, v = ((a @ w[(kind, layer)].T).reshape(n, -1, d) for kind in (syn.W_Q, syn.W_K, syn.W_V))
            cos, sin = (t[pos0:pos0 + n] for t in self.tables)
            q, k = O.rope(q, cos, sin), O.rope(k, cos, sin)
            cache = self.caches[layer]
            cache.write(0, pos0, {"k": k.astype(np.float32), "v": v.astype(np.float32)})
            got = [engine.cache_rows(0, layer, which, pos0 + n).astype(np.float64) for which in (0, 1)]
            t = np.arange(pos0 + n)
            for name, rows in zip("kv", got):
                for g in range(kv):
                    step = cache.s[name][0, g, t // cache.block].astype(np.float64)[:, None]
                    off = np.abs(rows[:, g] - cache.value(name, 0, g, t)) / step
                    assert off.max() < 1.001 and (off > 0.01).mean() < 0.01, (layer, name, off.max(), (off > 0.01).mean())
            out = np.zeros((n, heads, d))
            for i in range(n):
                see = O.visible(pos0 + i, self.window, self.sinks)
                for h in range(heads):
                    g = h // (heads // kv)
                    s = got[0][see, g] @ q[i, h] / np.sqrt(d)
                    p = np.exp(s - s.max())
                    out[i, h] = (p / p.sum()) @ got[1][see, g]
            x = x + out.reshape(n, -1) @ w[(syn.W_O, layer)].T
            a = self.norm(x, syn.W_POST_NORM, layer)
            gate, up = a @ w[(syn.W_GATE, layer)].T, a @ w[(syn.W_UP, layer)].T
            x = x + (gate / (1 + np.exp(-gate)) * up) @ w[(syn.W_DOWN, layer)].T
        return self.norm(x[-1], syn.W_FINAL_NORM, -1) @ w[(syn.W_LM_HEAD, -1)].T


def engine(cfg, weights):
    model = Llama(cfg)
    model.load_fp32(weights)
    return model


@pytest.mark.parametrize("cfg,block,window,sinks", [(CFG, 64, 0, 0), (CFG, 32, 40, 3), (WIDE, 128, 0, 0),
                                                    (WIDE, 64, 100, 1)])
def test_prompts_and_single_tokens(lib, cuda, cfg, block, window, sinks):
    weights = syn.llama_weights(cfg, 7, std=0.08)
    ids = syn.prompts(cfg, 1, 260, 3)[0]
    with engine(cfg, weights) as model:
        model.cache("int8", block, window, sinks)
        want = Model(cfg, weights, block, window, sinks)
        pos = 0
        for n in (70, 1, 1, 130, 5, 1):  # many rows, few rows and one
            model.forward_ids(ids[pos:pos + n], pos == 0)
            logits = want.forward(ids[pos:pos + n], pos, model)
            np.testing.assert_allclose(model.logits(), logits, rtol=1e-4, atol=1e-4 * np.abs(logits).max())
            pos += n


def test_int8_weights_and_int8_cache(lib, cuda):
    planes, dense = syn.llama_int8(CFG, 5)
    ids = syn.prompts(CFG, 1, 40, 4)[0]
    with Llama(CFG) as model:
        model.load_int8(planes, dense)
        model.cache()
        want = Model(CFG, dense, 64, 0, 0)
        for lo, hi in ((0, 30), (30, 31), (31, 40)):
            model.forward_ids(ids[lo:hi], lo == 0)
            logits = want.forward(ids[lo:hi], lo, model)
            np.testing.assert_allclose(model.logits(), logits, rtol=1e-4, atol=1e-4 * np.abs(logits).max())


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 4)])
def test_generate(lib, cuda, window, sinks):
    """Decoding through the captured step: in a batch as alone, ended by the
    context as the fp32 cache ends it, and each id the best or nearly so for a
    forward over all of the ids before it (its cache is quantised at once, not
    token by token: scales differ by a block's growth, logits by little)."""
    weights = syn.llama_weights(CFG, 9, std=0.08)
    prompts = [syn.prompts(CFG, 1, n, 30 + n)[0] for n in (1, 63, 64, 200)]
    with engine(CFG, weights) as model:
        model.cache("int8", 64, window, sinks)
        alone = [model.generate(p, 40) for p in prompts]
        for got, want in zip(model.generate_batch(prompts, 40), alone):
            assert np.array_equal(got, want)
        assert len(model.generate(prompts[3], 500)) == CFG["context"] - 200 + 1
        for p, out in zip(prompts, alone):
            assert len(out) == 40
            for n in (0, 1, 20, 39):
                model.forward_ids(np.concatenate([p, out[:n]]), True)
                logits = model.logits()
                assert logits.max() - logits[out[n]] <= 0.02 * (logits.max() - logits.min())


def test_switching_caches_keeps_the_fp32_results(lib, cuda):
    weights = syn.llama_weights(CFG, 9)
    prompt = syn.prompts(CFG, 1, 50, 2)[0]
    with engine(CFG, weights) as model:
        want = model.generate(prompt, 30)
        model.forward_ids(prompt, True)
        logits = model.logits()
        model.cache("int8", 32, 16, 2)
        model.generate(prompt, 30)
        model.cache("f32")
        assert np.array_equal(model.generate(prompt, 30), want)
        model.forward_ids(prompt, True)
        assert np.array_equal(model.logits(), logits)


@pytest.mark.parametrize("kind", ["f32", "int8"])
def test_generating_again_after_sequences_ended(lib, cuda, kind):
    """Sequences that ended (here by a full context) do not count towards the
    next call's, whose loop looks every 32 steps whether all have."""
    prompts = [syn.prompts(CFG, 1, n, n)[0] for n in (300, 310)]
    with engine(CFG, syn.llama_weights(CFG, 9, std=0.08)) as model:
        model.cache(kind)
        short = syn.prompts(CFG, 1, 20, 6)[0]
        want = model.generate(short, 100)
        assert [len(x) for x in model.generate_batch(prompts, 50)] == [21, 11]
        assert np.array_equal(model.generate(short, 100), want) and len(want) == 100


def test_refusals(lib, cuda):
    with engine(CFG, syn.llama_weights(CFG, 1)) as model:
        with pytest.raises(ValueError):
            model.cache("fp8")
        for kind, block, window, sinks in ((2, 64, 0, 0), (1, 16, 0, 0), (1, 0, 0, 0), (1, 64, -1, 0), (1, 64, 0, -1),
                                           (0, 0, 8, 0), (0, 0, 0, 1), (0, 64, 0, 0)):
            assert lib.accel_llama_cache(model._model, kind, block, window, sinks) == 1
            assert lib.accel_llama_last_error()
        assert len(model.generate(np.array([1, 2], np.int32), 4)) == 4  # the fp32 cache is still there
    assert lib.accel_llama_cache(None, 1, 64, 0, 0) == 1
    with Llama(syn.TINY_LLAMA) as tiny:  # heads of 16
        with pytest.raises(RuntimeError, match="head size"):
            tiny.cache()


def test_values_that_are_not_finite_fail_the_call(lib, cuda):
    weights = dict(syn.llama_weights(CFG, 1))
    embed = weights[(syn.W_EMBED, -1)].copy()
    embed[5] = np.inf
    weights[(syn.W_EMBED, -1)] = embed
    with engine(CFG, weights) as model:
        model.cache()
        good = model.generate(np.array([1, 2], np.int32), 1)
        with pytest.raises(RuntimeError, match="not finite"):
            model.generate(np.array([1, 5], np.int32), 4)
        with pytest.raises(RuntimeError, match="not finite"):
            model.forward_ids(np.array([5], np.int32), True)
        assert np.array_equal(model.generate(np.array([1, 2], np.int32), 1), good)
