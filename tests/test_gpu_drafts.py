"""examples/drafts.py on a B200: the paged cache, its attention, the probabilities and the verification of drafts together,
against the whole model's forward on the same seeded weights.

The two differ by the order of fp32 sums and the Q8 rounding of activations that follows from it: logprobs agree within
LP_TOL of tests/test_gpu_model.py, so a greedy choice must lie within twice that of the model's best."""
from __future__ import annotations

import importlib.util

import numpy as np
import pytest

from conftest import ROOT
from large_model_b200 import synth

pytestmark = pytest.mark.gpu
LP_TOL = 5e-3


@pytest.fixture(scope="module")
def drafts():
    spec = importlib.util.spec_from_file_location("drafts", ROOT / "examples" / "drafts.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def logprobs(x):
    x = x.astype(np.float64)
    return x - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)) - x.max(-1, keepdims=True)


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_greedy_with_drafts(cuda, drafts, kv):
    m, cfg = cuda, synth.MODEL_CONFIGS["tiny"]
    typ = m.T_F16 if kv == "f16" else m.T_F32
    model = drafts.PagedModel(cfg, 3, 64, 16, 256, typ)
    prompt = synth.random_ids(cfg.vocab, 37, 11)
    tails = [synth.random_ids(cfg.vocab, n, 20 + n) for n in (1, 4, 30)]
    plain, steps, made, _ = drafts.generate(model, prompt, tails, 12, draft=lambda b, known, n: [])
    assert steps == 12 and made == 0
    whole = m.Model.from_synth(cfg, 3, 256)
    whole.set_kv_type(typ)
    for ids, tail in zip(plain, tails):
        n0 = len(prompt) + len(tail)
        lp = logprobs(whole.forward(ids, 0, all_logits=True))
        for i in range(n0, len(ids)):
            assert lp[i - 1].max() - lp[i - 1][ids[i]] <= 2 * LP_TOL, (i, ids[i])
    whole.close()

    # guesses that are right stand, wrong ones fall, and the tokens stay the same (other batch shapes, so up to near ties)
    def right(b, known, n):
        return plain[b][len(known):len(known) + n] if known == plain[b][:len(known)] else []

    def second_wrong(b, known, n):
        g = right(b, known, n)
        return g[:1] + [(t + 1) % cfg.vocab for t in g[1:]]
    for how, most in ((right, 4), (second_wrong, 7)):
        got, steps, made, stood = drafts.generate(model, prompt, tails, 12, draft=how)
        for b in range(len(tails)):
            same = [x == y for x, y in zip(got[b], plain[b])]
            if not all(same):
                i = same.index(False)
                assert abs(lp_at(m, cfg, typ, plain[b][:i], (got[b][i], plain[b][i]))) <= 2 * LP_TOL, (b, i)
        if all(g == p for g, p in zip(got, plain)):
            assert steps <= most and (stood == made if how is right else 0 < stood < made)


def lp_at(m, cfg, typ, ids, pair):
    whole = m.Model.from_synth(cfg, 3, 256)
    whole.set_kv_type(typ)
    lp = logprobs(whole.forward(ids, 0))
    whole.close()
    return lp[pair[0]] - lp[pair[1]]


def test_sampled_is_reproducible(cuda, drafts):
    m, cfg = cuda, synth.MODEL_CONFIGS["tiny"]
    model = drafts.PagedModel(cfg, 3, 64, 16, 256)
    prompt, tails = synth.random_ids(cfg.vocab, 20, 1), [synth.random_ids(cfg.vocab, 3, 2)] * 2
    a = drafts.generate(model, prompt, tails, 10, temp=0.7, seed=4)
    assert a == drafts.generate(model, prompt, tails, 10, temp=0.7, seed=4)
    b = drafts.generate(model, prompt, tails, 10, temp=0.7, seed=5)[0]
    assert a[0] != b and all(0 <= t < cfg.vocab for k in a[0] + b for t in k)
    with pytest.raises(ValueError, match="too small"):
        drafts.generate(model, prompt, tails, 300)
