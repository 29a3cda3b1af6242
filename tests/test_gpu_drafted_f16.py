"""The operators of long contexts and drafted tokens together in f16, as examples/drafted_tokens.py uses them."""
import numpy as np
import pytest

from test_gpu_drafted_example import example  # noqa: F401 (a fixture)
from test_gpu_longctx import EPS16, f64

pytestmark = pytest.mark.gpu
MADE = dict(window=24, sinks=4, positions=120, rows_at_once=16)
TEXTS = [np.random.default_rng(6).integers(0, 512, n).tolist() for n in (1, 17, 70)]  # (the last one goes round the ring)


@pytest.mark.parametrize("cache", ["f16", "q4", "f32"])
@pytest.mark.parametrize("n", [1, 5, 16])
def test_f16_logits_are_those_of_f32(ctx, example, cache, n):  # noqa: F811
    logits = []
    for arithmetic in ("f32", "f16"):
        model, _ = example.models(ctx, len(TEXTS), 4, cache=cache, arithmetic=arithmetic, **MADE)
        model.read(TEXTS, 16)
        tokens = np.array([[t[-1], *range(1, n)] for t in TEXTS], np.int32)
        logits.append(model.forward(tokens, [len(t) - 1 for t in TEXTS]).to_numpy().astype(f64))
    want, got = logits
    # about 14 roundings to f16 per layer (weights, operands, results), five more at the end, independent of each other and of about
    # the stream's size each; six deviations.  Over 4 bits some codes are their neighbours, a fifteenth of a group's range away.
    tol = 6 * np.sqrt(3 * 14 + 5) * EPS16 if cache != "q4" else 0.25
    assert np.abs(got - want).max() <= tol * np.sqrt((want ** 2).mean())


@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_drafts_are_verified_in_f16(ctx, example, cache):  # noqa: F811
    made = dict(cache=cache, arithmetic="f16", **MADE)
    large, small = example.models(ctx, len(TEXTS), 4, **made)
    got, rounds, accepted = example.generate(ctx, large, small, TEXTS, 24, 4, 0.8, 1, 16)
    assert 0 < accepted and rounds <= 24
    for t, g in zip(TEXTS, got):
        assert g[:len(t)] == t and len(g) >= len(t) + 24 and all(0 <= x < 512 for x in g)
