"""The operators for many answers to one prompt at the ends of what their calls accept: temperatures and logits at the types' limits, batches of nothing but padding,
rows of padding that hold anything."""
import numpy as np
import pytest

import test_gpu_answers as base
from rllama_amd import Tensor
from test_gpu_answers import first_of_the_largest, logprobs_reference, shared_case, shared_reference
from test_gpu_longctx import EPS16, EPS32, INVALID, NUMPY, TYPES, f16, f32, f64, refused, upload, values

pytestmark = pytest.mark.gpu


# -- log probabilities --------------------------------------------------------------------------------------------------------------------

def check_logprobs(ctx, x, temperature, top=5):
    """All results of rows x against 64 bits.  An exponent is the difference of two logits (exact or rounded once) times 1 / temperature (rounded once); the weights' sum,
    all of them positive, and its logarithm add the rest, as in test_logprobs."""
    rows, vocab = x.shape
    top = min(top, vocab)
    ids = first_of_the_largest(x, vocab)
    tokens = np.ascontiguousarray(ids[:, [0, min(1, vocab - 1), vocab // 2, vocab - 1]])
    got = [t.to_numpy().astype(f64) for t in Tensor.from_numpy(ctx, x).token_logprobs(Tensor.from_numpy(ctx, tokens), temperature, top)]
    with np.errstate(over="ignore", invalid="ignore"):
        want, entropy = logprobs_reference(x, temperature)
        for g, w in ((got[0], np.take_along_axis(want, tokens, 1)), (got[3], np.take_along_axis(want, ids[:, :top], 1))):
            tol = EPS32 * (8 + 2 * np.sqrt(vocab) + 6 * np.abs(w) + 6 * np.log(vocab))
            assert not np.isnan(g).any()
            lost = w.astype(f32) == -np.inf  # (past what 32 bits hold)
            assert ((g == -np.inf) & lost | ~lost & (np.abs(g - w) <= tol)).all()
    assert (np.abs(got[1] - entropy) <= EPS32 * (16 + 2 * np.sqrt(vocab)) * (np.abs(entropy) + np.log(vocab) * (vocab > 1) * 8)).all()
    assert np.array_equal(got[2], ids[:, :top])


@pytest.mark.parametrize("temperature", [1e-30, 1e-12, 1e-9, 3e-9, 1e-8, 1e-7, 1e-6, 4e-5, 1e-3, 0.05, 1e3, 1e30])
@pytest.mark.parametrize("vocab", [33, 1000, 6000, 10000, 32000, 40000])
@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_logprobs_at_every_temperature(ctx, vocab, kind, temperature):
    """Rows whose largest entry is small, large, negative, the type's largest and smallest number and 0, alone and shared by several."""
    rng = np.random.default_rng(vocab)
    info = np.finfo(NUMPY[kind])
    x = np.concatenate([rng.standard_normal((3, vocab)) * 3, rng.standard_normal((3, vocab)) * 30, rng.standard_normal((2, vocab)) - 700, np.zeros((6, vocab))]).astype(NUMPY[kind])
    x[8:] = -np.abs(rng.standard_normal((6, vocab))) * 5
    x[8, 7], x[9, 9], x[10, 11], x[11, 3], x[12, 5] = info.max, info.max, info.tiny, info.smallest_subnormal if kind == "f16" else info.tiny, 0.0
    x[13] = info.min / 2
    for r, copies in ((1, 2), (4, 30), (7, 3), (9, 2), (10, 7), (12, 4)):  # ties
        x[r, rng.choice(vocab, copies, replace=False)] = x[r].max()
    check_logprobs(ctx, x, temperature)


@pytest.mark.parametrize("rows", [900])
@pytest.mark.parametrize("vocab", [6000, 10000, 32000])
def test_logprobs_of_many_rows_at_low_temperatures(ctx, rows, vocab):
    """The kernels for many rows."""
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(f16)
    x[::3, 17] = x[::3].max(1)
    for temperature in (1e-9, 1e-30):
        check_logprobs(ctx, x, temperature)


@pytest.mark.parametrize("vocab", [33, 6000, 32000, 40000])
@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_logprobs_of_logits_from_end_to_end(ctx, vocab, kind):
    """The type's largest and lowest number in one row: their difference is past what 32 bits hold, its quotient by a high temperature is not."""
    info = np.finfo(NUMPY[kind])
    x = np.zeros((5, vocab), NUMPY[kind])
    x[0, ::2], x[0, 1::2] = info.max, info.min
    x[1, 4:], x[1, 3] = info.min, info.max
    x[2, :], x[2, 30] = info.min, info.max
    x[3, :] = np.linspace(-1, 1, vocab) * f64(info.max)
    x[4, 1] = info.min
    for temperature in (1.0, 1e30, 2.5e29, 1e-30):
        check_logprobs(ctx, x, temperature)


def test_the_entropy_may_be_left_out(ctx):
    """entropy=False: None, and the library is not asked for it; a call that asks for nothing is refused."""
    logits, tokens = Tensor.from_numpy(ctx, np.eye(3, 50, dtype=f32)), Tensor.from_numpy(ctx, np.array([[0], [1], [2]], np.int32))
    whole = logits.token_logprobs(tokens, 0.5, 2)
    part = logits.token_logprobs(tokens, 0.5, 2, entropy=False)
    assert part[1] is None and whole[1].to_numpy().shape == (3, 1)
    assert all(np.array_equal(a.to_numpy(), b.to_numpy()) for a, b in zip(whole, part) if b is not None)
    assert logits.token_logprobs(entropy=whole[1])[1] is whole[1]
    refused(INVALID, logits.token_logprobs, entropy=False)


# -- attention: padding -------------------------------------------------------------------------------------------------------------------

IDLE = [
    # hd, heads, kv heads, rows of a text, prefix, texts
    (128, 32, 32, 20, 2000, 64), (128, 32, 8, 4, 300, 128), (64, 64, 8, 1, 1000, 128), (128, 40, 40, 16, 1000, 33), (128, 4, 4, 1, 100, 40), (32, 8, 1, 3, 128, 30), (128, 2, 2, 40, 17, 2),
]


@pytest.fixture(params=[None, "1", "2"])
def form(ctx, request):
    """The form that the estimate chooses, and either of the two."""
    ctx.set_option("ATTN_SHARED_FORM", request.param)
    yield ctx
    ctx.set_option("ATTN_SHARED_FORM", None)


@pytest.mark.parametrize("hd,H,G,n,P,B", IDLE)
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_an_idle_batch_behind_a_prefix(form, hd, H, G, n, P, B, cache):
    """Every text is padding: zeros, whatever the prefix's length and the number of rows."""
    rng = np.random.default_rng(P)
    pk, pv = (upload(form, rng.standard_normal((G * P, hd)), cache) for _ in range(2))
    own = upload(form, np.full((B * G * n, hd), np.nan), cache)
    q = Tensor.from_numpy(form, rng.standard_normal((B * n, H * hd)).astype(f16))
    for starts in ([-n] * B, [-n - b for b in range(B)]):
        out = Tensor.from_numpy(form, np.full((B * n, H * hd), np.nan, f16))
        q.attn_shared(pk, pv, P, own, own, H, G, n, starts, out=out)
        assert (out.to_numpy() == 0).all()


@pytest.mark.parametrize("hd,H,G,n,P,B", IDLE[4:])
def test_one_text_of_an_idle_batch(form, hd, H, G, n, P, B):
    starts = [-n] * (B - 1) + [1 - n]
    out, want, bound, _, _ = shared_case(form, hd, H, G, n, P, P, 40, starts, "f16", "f16")
    got = out.astype(f64).reshape(want.shape)
    assert (np.abs(got - want) <= bound).all() and (got[:-1] == 0).all() and (got[-1, -1] != 0).all()


@pytest.mark.parametrize("kind,cache", TYPES)
@pytest.mark.parametrize("hd,H,G,n,P,B", [(64, 4, 2, 1, 150, 5), (128, 8, 2, 3, 40, 9), (32, 6, 2, 1, 3000, 4), (64, 4, 4, 30, 700, 5), (128, 16, 2, 1, 900, 40), (64, 2, 1, 70, 60, 3), (128, 4, 1, 12, 0, 6)])
def test_padding_rows_hold_anything(form, hd, H, G, n, P, B, kind, cache):
    """Queries of padding rows are infinite, NaN, or the type's largest number, which overflows with any key: their results are zeros, and the other rows do not notice."""
    rng = np.random.default_rng(P + n)
    S = 90
    info = np.finfo(NUMPY[kind])
    starts = [0 if b % 3 == 0 else -n if b % 3 == 1 else -(n // 2) for b in range(B)]  # whole, idle, and padding in front
    q = rng.standard_normal((B, n, H, hd)).astype(NUMPY[kind])
    for b, start in enumerate(starts):
        for i in range(min(n, -start)):
            q[b, i, :, ::[1, hd][b % 2]] = [np.inf, -np.inf, np.nan, info.max, info.min][(b + i) % 5]  # (all dims, or the first alone: scores that are infinite, or not numbers)
            q[b, i, :, 1::2] *= [1, -1][i % 2]
    planes = [upload(form, rng.standard_normal((rows, hd)), cache) for rows in (G * max(P, 1), G * max(P, 1), B * G * S, B * G * S)]
    wide = [values(t).reshape(G, -1, hd)[:, :P] if i < 2 else values(t).reshape(B, G, S, hd) for i, t in enumerate(planes)]
    clean = q.astype(f64)
    for b, start in enumerate(starts):
        clean[b, :max(0, min(n, -start))] = 0
    want, bound = shared_reference(clean, *wide, starts)
    if kind == "f16":  # the result is rounded to f16; the weights may be
        bound = bound + 2 * EPS16 * max(np.abs(x).max() for x in (wide[1], wide[3]) if x.size)
    out = Tensor.from_numpy(form, np.full((B * n, H * hd), np.nan, NUMPY[kind]))
    Tensor.from_numpy(form, q.reshape(B * n, -1)).attn_shared(*planes[:2], P, *planes[2:], H, G, S, starts, out=out)
    got = out.to_numpy().astype(f64).reshape(want.shape)
    for b, start in enumerate(starts):
        assert (got[b, :max(0, min(n, -start))] == 0).all()
    assert (np.abs(got - want) <= bound).all()


# -- products -----------------------------------------------------------------------------------------------------------------------------

@pytest.fixture
def exact(ctx):
    ctx.set_option("GEMM_F8_EXACT", "1")
    yield ctx
    ctx.set_option("GEMM_F8_EXACT", None)


@pytest.mark.parametrize("m,n,k", base.PRODUCTS)
@pytest.mark.parametrize("source,spread", [("f16", 1.0), ("f8", 1.0), ("f8", 3.0)])
def test_f16_results_summed_up_in_f32_on_request(exact, m, n, k, source, spread):
    """Columns of x a few powers of ten apart, whose products the 8-bit instruction cuts off beside the largest ones: the bound is that of sums in f32, and the result's rounding."""
    rng = np.random.default_rng(m * 7 + n + k)
    x = (rng.standard_normal((m, k)) * np.exp(spread * rng.standard_normal((1, k)))).astype(f32)
    x = x / np.abs(x).max() * 100  # (within f16)
    w = Tensor.from_numpy(exact, (rng.standard_normal((n, k)) / np.sqrt(k)).astype(f32)).convert(base.TILES)
    x = Tensor.from_numpy(exact, x.astype(f16 if source == "f16" else f32))
    eight = x.convert(base.F8)
    a, b = base.stands_for(*base.parts(eight), False), base.stands_for(*base.parts(w), True)
    out = Tensor.from_numpy(exact, np.full((m, n), np.nan, f16))
    (eight if source == "f8" else x).matrix_mul_f8(w, out=out)
    want = a @ b.T
    assert (np.abs(out.to_numpy() - want) <= base.product_bound(a, b, k, "f32") + EPS16 * np.abs(want) + 2.0 ** -25).all()
