"""The operators of long contexts and drafted tokens together, as examples/drafted_tokens.py uses them."""
import importlib.util
import os

import numpy as np
import pytest

from rllama_amd import Context

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "drafted_tokens.py")


@pytest.fixture(scope="module")
def ctx():
    return Context(0)


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("drafted_tokens", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cache", ["f32", "f16", "q4"])
def test_drafts_do_not_change_the_greedy_text(ctx, example, cache):
    chats, k, rows, new, window = 3, 4, 16, 40, 24
    rng = np.random.default_rng(5)
    texts = [rng.integers(0, 512, n).tolist() for n in (1, 17, 50)]  # (the last one is longer than the window)
    made = dict(window=window, sinks=4, positions=120, rows_at_once=rows, cache=cache)
    large, small = example.models(ctx, chats, k, **made)
    got, rounds, accepted = example.generate(ctx, large, small, texts, new, k, 0.0, 1, rows)
    assert 0 < accepted and rounds <= chats * new
    alone, _ = example.models(ctx, chats, k, **made)
    alone.read(texts, rows)
    want = [list(t) for t in texts]
    for _ in range(new):
        probs = alone.forward(np.array([[t[-1]] for t in want], np.int32), [len(t) - 1 for t in want]).softmax_rows(0.0).to_numpy()
        assert (probs.sum(1) == 1).all()
        for t, p in zip(want, probs):
            t.append(int(p.argmax()))
    for g, w in zip(got, want):
        assert len(g) >= len(w) and g[:len(w)] == w


def test_a_draft_by_the_model_itself_is_always_accepted(ctx, example):
    chats, k, rows = 2, 3, 8
    texts = [[5, 6, 7], [9, 8, 7, 6, 5, 4, 3, 2, 1, 0, 11]]
    large, _ = example.models(ctx, chats, k, window=20, sinks=2, positions=100, rows_at_once=rows, cache="f32")
    same, _ = example.models(ctx, chats, k, window=20, sinks=2, positions=100, rows_at_once=rows, cache="f32")
    _, rounds, accepted = example.generate(ctx, large, same, texts, 32, k, 0.7, 3, rows)
    # (p and q of one row differ by roundings only: a refusal needs a variate that falls between them)
    assert rounds == 8 and accepted == rounds * chats * k
