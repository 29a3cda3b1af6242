"""The operators for long contexts and drafted tokens against their definitions in 64 bits: tensors of 4 bits, the append of a
projection's rows to the caches, attention with a window over caches of 16, 32 and 4 bits, probabilities of rows and the verification of
drafts; their special rows (padding, empty masks, NaN in what nobody sees, rings), their refusals, memory of other owners and streams."""
import os
import subprocess
import sys

import numpy as np
import pytest

import rllama_amd
from rllama_amd import RllamaHipError, Tensor, TensorDType

pytestmark = pytest.mark.gpu
f16, f32, f64 = np.float16, np.float32, np.float64
EPS32, EPS16 = 2.0 ** -24, 2.0 ** -11  # half a unit in the last place, relative
DTYPE = {"f16": TensorDType.Float16, "f32": TensorDType.Float32, "q4": TensorDType.K4BitQuantization}
NUMPY = {"f16": f16, "f32": f32}


# -- 4 bits ----------------------------------------------------------------------------------------------------------------------

def q4_encode(x):
    """The buffer of an array [rows x cols], by the definition: every step is one operation in 32 bits."""
    rows, cols = x.shape
    g = x.astype(f32).reshape(rows, cols // 32, 32)
    with np.errstate(all="ignore"):
        low = (np.nanmin(np.where(np.isnan(g), np.inf, g), -1) + f32(0)).astype(f16)  # (a zero is positive)
        scale = ((np.nanmax(np.where(np.isnan(g), -np.inf, g), -1) - low.astype(f32) + f32(0)) / f32(15)).astype(f16)
        broken = ~(np.isfinite(g).all(-1) & np.isfinite(low) & np.isfinite(scale))
        s = scale.astype(f32)[..., None]
        code = np.clip(np.rint((g - low.astype(f32)[..., None]) / s), 0, 15)
    code = np.where((s > 0) & ~broken[..., None], code, 0).astype(np.uint8).reshape(rows, cols // 2, 2)
    pairs = np.stack([scale.view(np.uint16), low.view(np.uint16)], -1)
    pairs[broken] = (0, 0x7e00)
    return np.concatenate([(code[..., 0] | code[..., 1] << 4).reshape(-1), pairs.reshape(-1).view(np.uint8)])


def q4_decode(buffer, rows, cols):
    count = rows * cols
    b = buffer[:count // 2]
    code = np.stack([b & 15, b >> 4], -1).reshape(rows, cols // 32, 32).astype(f64)
    pairs = buffer[count // 2:].view(f16).reshape(rows, cols // 32, 2).astype(f64)
    return (pairs[..., 1:] + code * pairs[..., :1]).reshape(rows, cols)


def upload(ctx, x, kind):
    t = Tensor.from_numpy(ctx, x.astype(f32 if kind == "q4" else NUMPY[kind]))
    return t.convert(TensorDType.K4BitQuantization) if kind == "q4" else t


def values(t):
    """What a tensor of any type holds, in 64 bits."""
    if t.dtype() == TensorDType.K4BitQuantization:
        return q4_decode(t.to_numpy(), t.rows(), t.cols())
    return t.to_numpy().astype(f64)


def special_values(rng, rows, cols):
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-9, 6, (rows, 1)))).astype(f32)
    x[0, 3] = np.nan
    x[1, 40] = np.inf
    x[2, 0] = -np.inf
    x[3, 5] = 1e6            # its scale fits f16, nothing else
    x[4, 7] = -1e6           # lowest does not
    x[5, :32] = 0.37         # one value: scale 0
    x[6, :] *= 1e-7          # scale below f16's smallest
    x[7, :32] = 0.0
    x[8, :32] = np.linspace(-7.5, 7.5, 32)  # ties
    return x


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_conversion_to_and_from_4_bits_is_its_definition(ctx, kind):
    rng = np.random.default_rng(5)
    with np.errstate(over="ignore"):
        x = special_values(rng, 37, 96).astype(NUMPY[kind])
    t = Tensor.from_numpy(ctx, x).convert(TensorDType.K4BitQuantization)
    want = q4_encode(x)
    assert np.array_equal(t.to_numpy(), want)
    back = t.convert(TensorDType.Float32).to_numpy()
    assert np.array_equal(back, q4_decode(want, 37, 96).astype(f32), equal_nan=True)
    with np.errstate(over="ignore"):
        assert np.array_equal(t.convert(TensorDType.Float16).to_numpy(), back.astype(f16), equal_nan=True)
    assert np.isnan(back[0, :32]).all() and np.isfinite(back[0, 32:]).all() and np.isnan(back[1, 32:64]).all() and np.isnan(back[4, :32]).all()
    assert np.isfinite(back[5:]).all()
    copy = t.clone()
    assert copy.dtype() == TensorDType.K4BitQuantization and np.array_equal(copy.to_numpy(), want)
    if kind == "f16":
        assert np.array_equal(Tensor.from_numpy(ctx, x).convert(TensorDType.Float32).to_numpy(), x.astype(f32), equal_nan=True)


# -- append ------------------------------------------------------------------------------------------------------------------------

def rotation(positions, hd, theta=10000.0):
    return np.outer(positions, theta ** (-np.arange(0, hd, 2) / hd))


def append_reference(qkv, H, G, hd, positions, qn, kn, eps, halves):
    x = qkv.astype(f64).reshape(len(positions), H + 2 * G, hd)
    a = rotation(positions, hd).astype(f64)
    c, s = np.cos(a).astype(f32).astype(f64)[:, None], np.sin(a).astype(f32).astype(f64)[:, None]
    out = x.copy()
    for lo, hi, w in ((0, H, qn), (H, H + G, kn)):
        y = x[:, lo:hi]
        if w is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(f64)
        re, im = (y[..., :hd // 2], y[..., hd // 2:]) if halves else (y[..., 0::2], y[..., 1::2])
        z = (re * c - im * s, re * s + im * c)
        out[:, lo:hi] = np.concatenate(z, -1) if halves else np.stack(z, -1).reshape(y.shape)
    return out[:, :H], out[:, H:H + G], out[:, H + G:]


def ring_row(t, S, sinks):
    return t if t < S else sinks + (t - sinks) % (S - sinks)


APPEND = [
    # hd, heads, kv heads, n, max_seq_len, sinks, positions of the first rows
    (128, 4, 4, 1, 40, 0, [17]),
    (128, 7, 1, 9, 40, 0, [0]),
    (64, 6, 2, 5, 33, 0, [3, 28, -2, -5]),     # the third one starts with padding, the fourth is idle
    (32, 2, 2, 67, 90, 0, [11, 0]),
    (64, 8, 8, 6, 24, 4, [20, 2000, 3]),       # a ring: the first one passes the end, the second is far behind it
]


@pytest.mark.parametrize("hd,H,G,n,S,sinks,starts", APPEND)
@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4"), ("f32", "f32"), ("f32", "q4"), ("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("halves,norms", [(False, True), (True, True), (False, False)])
def test_append(ctx, hd, H, G, n, S, sinks, starts, kind, cache, halves, norms):
    rng = np.random.default_rng(hd + 3 * H + n)
    B = len(starts)
    qkv = (rng.standard_normal((B * n, (H + 2 * G) * hd)) * 1.7).astype(NUMPY[kind])
    qn, kn = (rng.uniform(0.5, 1.5, (1, hd)).astype(f32) for _ in range(2))
    old_k, old_v = (rng.standard_normal((B * G * S, hd)) for _ in range(2))
    ck, cv = upload(ctx, old_k, cache), upload(ctx, old_v, cache)
    before = values(ck), values(cv)
    freqs = Tensor.zeros(ctx, 2100, hd, TensorDType.Float32).rope_table()
    q = Tensor.from_numpy(ctx, np.full((B * n, H * hd), np.nan, NUMPY[kind]))
    up = lambda w: Tensor.from_numpy(ctx, w) if norms else None  # noqa: E731
    Tensor.from_numpy(ctx, qkv).qkv_append(q, ck, cv, freqs, H, G, S, starts, q_norm=up(qn), k_norm=up(kn), eps=1e-5, halves=halves, sinks=sinks)
    got_q = q.to_numpy().astype(f64).reshape(B, n, H, hd)
    got = [x.reshape(B, G, S, hd) for x in (values(ck), values(cv))]
    want = [x.reshape(B, G, S, hd).copy() for x in before]
    written = np.zeros((B, G, S), bool)
    # norm, weight and rotation: a sum of hd squares (its error halves under the root) and about 8 roundings of values up to sqrt(2) max|y|
    tol32 = (np.sqrt(hd) + 12) * EPS32
    for b, start in enumerate(starts):
        pos = np.arange(start, start + n)
        rq, rk, rv = append_reference(qkv.reshape(B, n, -1)[b], H, G, hd, np.maximum(pos, 0), qn if norms else None, kn if norms else None, 1e-5, halves)
        rq[pos < 0] = 0
        top = np.abs(rq).max() + 1e-30
        assert np.abs(got_q[b] - rq).max() <= (tol32 + (EPS16 if kind == "f16" else 0)) * top
        assert (got_q[b][pos < 0] == 0).all()
        for i, p in enumerate(pos):
            if p < 0:
                continue
            row = ring_row(p, S, sinks)
            written[b, :, row] = True
            for which, r in ((0, rk[i]), (1, rv[i])):
                want[which][b, :, row] = r
    for which in range(2):
        w, g = want[which], got[which]
        assert np.array_equal(g[~written], w[~written])  # nothing else is touched
        w, g = w[written], g[written]
        top = np.abs(w).max()
        if cache == "q4":
            grp = w.reshape(len(w), -1, 32)
            lo, hi = grp.min(-1, keepdims=True), grp.max(-1, keepdims=True)
            # half a step, the step's and the lowest value's own rounding (over at most 15 steps), and what the value came with
            tol = (hi - lo) / 15 * (0.5 + 16 * EPS16) + 3 * EPS16 * np.abs(lo) + 2 * tol32 * top + 2.0 ** -24
            assert (np.abs(g.reshape(grp.shape) - grp) <= tol).all()
        else:
            assert np.abs(g - w).max() <= (tol32 + (EPS16 if cache == "f16" else 0)) * top


def test_append_writes_what_the_token_step_writes(ctx):
    """Without norms, one row: bit for bit the queries and cache rows of the forward's own rotation and cache write."""
    rng = np.random.default_rng(2)
    H, hd, S, pos = 3, 64, 50, 37
    x = rng.standard_normal((3, H * hd)).astype(f32)
    freqs = Tensor.zeros(ctx, S, hd, TensorDType.Float32).rope_table()
    a = [Tensor.zeros(ctx, H * S, hd, TensorDType.Float16) for _ in range(4)]
    q, k, v = (Tensor.from_numpy(ctx, r.reshape(1, -1)) for r in x)
    q.rope_kvwrite(k, v, a[0], a[1], H, S, pos)
    q2 = Tensor.zeros(ctx, 1, H * hd, TensorDType.Float32)
    Tensor.from_numpy(ctx, x.reshape(1, -1)).qkv_append(q2, a[2], a[3], freqs, H, H, S, [pos])
    assert np.array_equal(q.to_numpy(), q2.to_numpy())
    assert np.array_equal(a[0].to_numpy(), a[2].to_numpy()) and np.array_equal(a[1].to_numpy(), a[3].to_numpy())


# -- attention ------------------------------------------------------------------------------------------------------------------------

def seen_positions(p, window, sinks):
    t = np.arange(p + 1)
    return t[(t < sinks) | (t > p - window)] if window else t


def attention_reference(q, K, V, H, G, hd, starts, n, S, window, sinks):
    """q [B, n, H, hd], K and V [B, G, S, hd] in 64 bits; also the bound of the error that f32 arithmetic may leave and the largest
    sqrt(sum (q k)^2 / hd) of a seen pair, per row and head."""
    B = len(starts)
    out, bound, spread = np.zeros((B, n, H, hd)), np.zeros((B, n, H, 1)), np.zeros((B, n, H, 1))
    for b, start in enumerate(starts):
        for i in range(n):
            p = start + i
            if p < 0:
                continue
            t = seen_positions(p, window, sinks)
            rows = np.array([ring_row(int(x), S, sinks) for x in t]) if p >= S else t
            for g in range(G):
                k, v = K[b, g, rows], V[b, g, rows]
                hs = slice(g * (H // G), (g + 1) * (H // G))
                s = q[b, i, hs] @ k.T / np.sqrt(hd)
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[b, i, hs] = w @ v
                # a score is off by some roundings of a sum of hd terms, each weight by as much, the sums over t by theirs
                size = (np.abs(q[b, i, hs]) @ np.abs(k).T).max(-1, keepdims=True) / np.sqrt(hd)
                delta = 4 * np.sqrt(hd) * EPS32 * size
                bound[b, i, hs] = np.abs(v).max() * (2 * delta + (4 * np.sqrt(len(t)) + 16) * EPS32)
                spread[b, i, hs] = np.sqrt((q[b, i, hs] ** 2) @ (k ** 2).T / hd).max(-1, keepdims=True)
    return out, bound, spread


ATTEND = [
    # hd, heads, kv heads, n, max_seq_len, window, sinks, positions of the first rows
    (128, 4, 4, 1, 70, 0, 0, [0]),
    (128, 4, 4, 1, 70, 0, 0, [69]),
    (64, 2, 2, 1, 300, 0, 0, [255, 16, 31, 32, 0, -1]),
    (32, 8, 2, 1, 1200, 0, 0, [1000, 1199]),
    (128, 16, 1, 1, 2100, 0, 0, [2055]),
    (128, 34, 2, 1, 400, 0, 0, [333]),             # 17 heads share a key head
    (128, 8, 1, 5, 777, 0, 0, [700]),              # 40 rows on one key head
    (64, 7, 7, 3, 150, 0, 0, [100, -2, -3, 0]),    # padding in front, an idle slot
    (64, 4, 2, 33, 64, 0, 0, [0]),
    (128, 2, 1, 130, 200, 0, 0, [0, 57, -40]),
    (32, 3, 3, 71, 400, 0, 0, [300]),
    (128, 3, 3, 257, 700, 0, 0, [431]),
    (128, 4, 2, 1, 600, 1, 0, [500]),              # a window of the row itself
    (128, 4, 2, 1, 600, 16, 4, [500, 3, 19]),
    (64, 4, 4, 1, 900, 100, 70, [850]),            # more first tokens than a tile
    (128, 4, 2, 6, 600, 33, 1, [500, 30]),
    (64, 2, 1, 150, 900, 64, 4, [600]),
    (128, 4, 1, 140, 500, 97, 3, [0]),
    (128, 2, 2, 200, 500, 300, 16, [100]),
    (32, 4, 2, 300, 700, 5, 40, [333]),
    (64, 4, 2, 1, 80, 40, 4, [79, 80, 5000, 117]), # rings
    (128, 4, 2, 7, 64, 50, 8, [60, 64, 1001]),
    (128, 2, 1, 90, 300, 130, 4, [250, 7777]),
    (32, 2, 2, 1, 50, 49, 0, [99]),
]
MANY_ROWS = [  # (two forms of the product: up to 256 workgroups, with uneven work up to 512, and above)
    (128, 20, 20, 260, 300, 0, 0, [0, 5, 40, -7, 0, 0, 0, 0, 0]),
    (64, 60, 20, 130, 330, 70, 3, [190, 200, -129, 3]),
    (32, 30, 30, 129, 200, 60, 5, [0, 180, 400, 31, 64, 71, 1000, 70, 69, 68]),
    (128, 24, 24, 129, 450, 200, 70, [300, 5000, 321, 440, 449, 448]),
    (128, 24, 24, 150, 700, 0, 0, [500, 550, 63, 64, 150, 300]),
    (64, 24, 24, 150, 700, 0, 0, [500, 550, 63, 64, 150, 300]),
    (32, 16, 16, 400, 400, 0, 0, [0, 0, 0]),
    (128, 8, 2, 40, 16100, 0, 0, [16000]),         # few of them behind long texts: cut into pieces
    (64, 4, 2, 90, 30100, 0, 0, [30010, -20]),
    (32, 4, 2, 100, 25200, 25000, 7, [30190]),
    (128, 40, 10, 140, 500, 97, 3, [0, 100, 333, 20]),
    (32, 40, 20, 300, 700, 5, 40, [333, 0]),
    (64, 36, 12, 150, 900, 64, 4, [600, 88, 3]),
]
TYPES = [("f16", "f16"), ("f16", "q4"), ("f32", "f32"), ("f32", "q4"), ("f32", "f16"), ("f16", "f32")]


def _attend_case(hd, H, G, n, S, window, sinks, starts, seed=0, poison=True):
    rng = np.random.default_rng(hd * 31 + H * 7 + n + S + seed)
    B = len(starts)
    q = rng.standard_normal((B, n, H, hd)) * 1.5
    K, V = rng.standard_normal((B, G, S, hd)), rng.standard_normal((B, G, S, hd))
    if poison:  # what no row sees holds NaN
        for b, start in enumerate(starts):
            keep = np.zeros(S, bool)
            for p in range(max(0, start), start + n):
                keep[[ring_row(int(t), S, sinks) for t in seen_positions(p, window, sinks)]] = True
            K[b, :, ~keep] = np.nan
            V[b, :, ~keep] = np.nan
    return q, K, V


@pytest.mark.parametrize("hd,H,G,n,S,window,sinks,starts", MANY_ROWS)
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_attention_of_many_rows(ctx, hd, H, G, n, S, window, sinks, starts, cache):
    test_attention(ctx, hd, H, G, n, S, window, sinks, starts, "f16", cache)


@pytest.mark.parametrize("hd,H,G,n,S,window,sinks,starts", ATTEND)
@pytest.mark.parametrize("kind,cache", TYPES)
def test_attention(ctx, hd, H, G, n, S, window, sinks, starts, kind, cache):
    B = len(starts)
    q, K, V = _attend_case(hd, H, G, n, S, window, sinks, starts)
    q = q.astype(NUMPY[kind]).astype(f64)
    ck, cv = upload(ctx, K.reshape(-1, hd), cache), upload(ctx, V.reshape(-1, hd), cache)
    K, V = (values(t).reshape(B, G, S, hd) for t in (ck, cv))
    want, bound, spread = attention_reference(q, K, V, H, G, hd, starts, n, S, window, sinks)
    Q = Tensor.from_numpy(ctx, q.reshape(B * n, H * hd).astype(NUMPY[kind]))
    out = Tensor.from_numpy(ctx, np.full((B * n, H * hd), np.nan, NUMPY[kind]))
    Q.attn_window(ck, cv, H, G, S, starts, window=window, sinks=sinks, out=out)
    got = out.to_numpy().astype(f64).reshape(B, n, H, hd)
    tol = bound
    if kind == "f16":
        top = np.nanmax(np.abs(V))
        # weights and result are rounded to f16; so are cached values that f16 does not hold, which moves a score by a sum of hd
        # independent roundings (four deviations are allowed)
        tol = tol + 2 * EPS16 * top
        if cache != "f16":
            tol = tol + EPS16 * top + 2 * top * 4 * (EPS16 / np.sqrt(3)) * spread
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / np.maximum(tol, 1e-30))
    assert worst.max() <= 1, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))
    for b, start in enumerate(starts):
        assert (got[b, :max(0, min(n, -start))] == 0).all()
    # the same again: no sum depends on which workgroup came first
    out2 = Tensor.zeros(ctx, B * n, H * hd, DTYPE[kind])
    Q.attn_window(ck, cv, H, G, S, starts, window=window, sinks=sinks, out=out2)
    assert np.array_equal(out2.to_numpy(), out.to_numpy())


@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4"), ("f32", "f32")])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1023, 1025, 3000])
def test_single_tokens_of_every_length(ctx, kind, cache, T):
    """Around every edge at which a sequence could be cut."""
    H, G, hd, S = 4, 2, 128, 3001
    q, K, V = _attend_case(hd, H, G, 1, S, 0, 0, [T - 1], seed=T)
    q = q.astype(NUMPY[kind]).astype(f64)
    ck, cv = upload(ctx, K.reshape(-1, hd), cache), upload(ctx, V.reshape(-1, hd), cache)
    K, V = (values(t).reshape(1, G, S, hd) for t in (ck, cv))
    want, bound, spread = attention_reference(q, K, V, H, G, hd, [T - 1], 1, S, 0, 0)
    got = Tensor.from_numpy(ctx, q.reshape(1, -1).astype(NUMPY[kind])).attn_window(ck, cv, H, G, S, [T - 1]).to_numpy().astype(f64).reshape(want.shape)
    top = np.nanmax(np.abs(V))
    tol = bound + (2 * EPS16 * top if kind == "f16" else 0) + (EPS16 * top + 2 * top * 4 * (EPS16 / np.sqrt(3)) * spread if cache == "q4" else 0)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 40])
def test_scores_far_apart(ctx, kind, n):
    """Scores of several hundred, rising and falling along the text: the running maximum moves all the time, weights underflow."""
    rng = np.random.default_rng(9)
    H, hd, S = 2, 64, 500
    start = S - n
    for order in (1, -1, 0):
        K = rng.standard_normal((1, H, S, hd)) * 0.1
        ramp = np.linspace(-40, 40, S) * order if order else rng.permutation(np.linspace(-40, 40, S))
        K[..., 0] = ramp
        q = rng.standard_normal((1, n, H, hd))
        q[..., 0] = 60.0  # scores from -300 to 300
        V = rng.standard_normal((1, H, S, hd))
        q, K, V = (x.astype(NUMPY[kind]).astype(f64) for x in (q, K, V))
        want, bound, _ = attention_reference(q, K, V, H, H, hd, [start], n, S, 0, 0)
        got = Tensor.from_numpy(ctx, q.reshape(n, -1).astype(NUMPY[kind])).attn_window(
            upload(ctx, K.reshape(-1, hd), kind), upload(ctx, V.reshape(-1, hd), kind), H, H, S, [start]).to_numpy().astype(f64).reshape(want.shape)
        # near the top a score of 300 has a unit of 2^-15 in f32: exp's argument is off by as much whatever the operands' type
        tol = bound + 2 * np.abs(V).max() * 300 * 4 * EPS32 + (2 * EPS16 * np.abs(V).max() if kind == "f16" else 0)
        assert (np.abs(got - want) <= tol).all()


def test_values_that_are_not_finite_reach_the_rows_that_see_them(ctx):
    H, hd, S, n = 1, 64, 64, 40
    rng = np.random.default_rng(1)
    for kind in ("f16", "f32"):
        K, V = rng.standard_normal((S, hd)), rng.standard_normal((S, hd))
        V[20, 5] = np.nan
        q = rng.standard_normal((n, hd)).astype(NUMPY[kind])
        got = Tensor.from_numpy(ctx, q).attn_window(upload(ctx, K, kind), upload(ctx, V, kind), H, H, S, [0]).to_numpy()
        assert np.isnan(got[20:, 5]).all()
        assert np.isfinite(got[:20]).all() and np.isfinite(np.delete(got, 5, 1)).all()


@pytest.mark.parametrize("n,start,H,B", [(40, 90, 1, 1), (90, 0, 2, 1), (300, 100, 2, 1), (130, 60, 20, 10), (130, 260, 30, 10)])
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_an_infinite_value_reaches_all_that_see_it_and_no_others(ctx, cache, n, start, H, B):
    hd, S = 32, start + n
    rng = np.random.default_rng(n)
    q = rng.standard_normal((B, n, H, hd))
    K, V = rng.standard_normal((B, H, S, hd)), rng.standard_normal((B, H, S, hd))
    at = min(70, S - 1)
    V[:, 0, at, 5] = np.inf  # (of 4 bits its whole group is NaN)
    got = Tensor.from_numpy(ctx, q.reshape(B * n, H * hd).astype(f16)).attn_window(upload(ctx, K.reshape(-1, hd), cache), upload(ctx, V.reshape(-1, hd), cache), H, H, S, [start] * B)
    got = got.to_numpy().reshape(B, n, H, hd)
    first = max(0, at - start)
    hit = got[:, first:, 0]
    if cache == "f16":
        assert (hit[..., 5] == np.inf).all() and np.isfinite(np.delete(hit, 5, -1)).all()
    else:
        assert np.isnan(hit).all()
    assert np.isfinite(got[:, :first]).all() and np.isfinite(got[:, :, 1:]).all()


@pytest.mark.parametrize("n", [1, 33])
def test_offsets_past_32_bits(ctx, n):
    """Planes of more than 2^32 elements: the last sequence's last rows."""
    B, hd, S, window = 4, 128, (1 << 23) + 1024, 50
    rng = np.random.default_rng(3)
    ck, cv = (Tensor.zeros(ctx, B * S, hd, TensorDType.Float16) for _ in range(2))
    freqs = Tensor.zeros(ctx, S, hd, TensorDType.Float32)  # no rotation: cos 0 would clear the keys, so they are written unrotated below
    try:
        start = S - n - window
        rows = n + window
        ones = np.zeros((1, hd), f32)
        ones[0, 0::2] = 1.0
        # the angles of the rows that are written: a table of zeros but for them
        tail = Tensor.from_device(ctx, _pointer(freqs) + start * hd * 4, rows, hd, TensorDType.Float32)
        up = Tensor.from_numpy(ctx, np.repeat(ones, rows, 0))
        rllama_amd._lib.check(ctx._lib.rlh_copy_inplace(tail._h, up._h))
        x = rng.standard_normal((B * rows, 3 * hd)).astype(f16)
        q = Tensor.zeros(ctx, B * rows, hd, TensorDType.Float16)
        starts = [-rows] * (B - 1) + [start]
        Tensor.from_numpy(ctx, x).qkv_append(q, ck, cv, freqs, 1, 1, S, starts)
        last = x.reshape(B, rows, 3, hd)[-1].astype(f64)
        assert np.array_equal(q.to_numpy().reshape(B, rows, hd)[-1], last[:, 0].astype(f16))
        qq = np.zeros((B, n, hd), f16)
        qq[-1] = last[window:, 0].astype(f16)
        got = Tensor.from_numpy(ctx, qq.reshape(B * n, hd)).attn_window(ck, cv, 1, 1, S, [-n] * (B - 1) + [start + window], window=window).to_numpy()
        for i in range(n):
            k, v = last[i + 1:i + window + 1, 1], last[i + 1:i + window + 1, 2]
            s = last[i + window, 0] @ k.T / np.sqrt(hd)
            w = np.exp(s - s.max())
            assert np.abs(got.reshape(B, n, hd)[-1, i] - w @ v / w.sum()).max() <= 3 * EPS16 * np.abs(v).max()
        assert (got.reshape(B, n, hd)[:-1] == 0).all()
    finally:
        for t in (ck, cv, freqs):
            t.free()


def _pointer(t):
    """A tensor's device address (the handle's second word)."""
    import ctypes as C
    return C.cast(t._h, C.POINTER(C.c_void_p))[1]


# -- probabilities ----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("vocab", [1, 3, 63, 64, 65, 1000, 1023, 4097, 32000, 32001, 50257, 131075])
@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_probabilities(ctx, vocab, kind, temperature):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((3, vocab)) * 4).astype(NUMPY[kind])
    x[1, ::2] = -np.inf if vocab > 1 else x[1, ::2]
    got = Tensor.from_numpy(ctx, x).softmax_rows(temperature).to_numpy().astype(f64)
    z = x.astype(f64) / temperature
    want = np.exp(z - z.max(-1, keepdims=True))
    want /= want.sum(-1, keepdims=True)
    # the argument of exp is off by a few roundings of up to 40 / temperature, the sum by its additions
    tol = want * (6 * EPS32 * 40 / temperature + (8 + 2 * np.sqrt(vocab)) * EPS32) + 1e-38
    assert (np.abs(got - want) <= tol).all()


def test_probabilities_of_special_rows(ctx):
    x = np.zeros((8, 700), f32)
    x[0] = -np.inf
    x[1, 5] = np.nan
    x[2, 699] = np.inf
    x[3] = -np.inf
    x[3, 13] = -3e38
    x[4] = 3e38
    x[5, [7, 9, 600]] = 2.0
    x[6] = np.finfo(f32).min
    x[7, 1] = -np.inf
    p = Tensor.from_numpy(ctx, x).softmax_rows(0.5).to_numpy()
    assert (p[0] == 0).all() and np.isnan(p[1]).all() and np.isnan(p[2]).all()
    assert p[3, 13] == 1 and p[3].sum() == 1
    assert np.allclose(p[4], 1 / 700, rtol=1e-6) and np.allclose(p[6], 1 / 700, rtol=1e-6)
    assert p[7, 1] == 0 and np.allclose(np.delete(p[7], 1), 1 / 699, rtol=1e-6)
    for t in (0.0, 1e-45):
        p = Tensor.from_numpy(ctx, x).softmax_rows(t).to_numpy()
        assert (p[0] == 0).all() and np.isnan(p[1]).all() and np.isnan(p[2]).all()
        for row, first in ((3, 13), (4, 0), (5, 7), (6, 0), (7, 0)):
            assert p[row, first] == 1 and p[row].sum() == 1
    tiny = Tensor.from_numpy(ctx, x[5:6]).softmax_rows(1e-30).to_numpy()
    assert np.allclose(tiny[0, [7, 9, 600]], 1 / 3, rtol=1e-6) and tiny.sum() == pytest.approx(1)


# -- verification -----------------------------------------------------------------------------------------------------------------------

def verify_reference(target, draft, drafted, uniforms):
    """By the definition, in whole numbers."""
    B, k = drafted.shape
    V = target.shape[1]
    out = np.full((B, k + 2), -1, np.int32)
    for b in range(B):
        count, take = 0, None
        while count < k:
            x = int(drafted[b, count])
            if not 0 <= x < V:
                break
            p = target[b * (k + 1) + count]
            q = f32(1) if draft is None else draft[b * k + count, x]
            if uniforms[b, count] * q < p[x]:
                out[b, 1 + count] = x
                count += 1
                continue
            take = np.zeros(V, f32) if draft is None else draft[b * k + count]
            if draft is None:
                take[x] = 1
            break
        p = target[b * (k + 1) + count]
        pick = -1
        for w in ([p - take] if take is not None else []) + [p]:
            with np.errstate(invalid="ignore"):
                w = np.nan_to_num(np.minimum(np.fmax(w, f32(0)), f32(1)), nan=0.0)
            units = [int(v) for v in np.rint(w * f32(2.0 ** 31)).astype(np.int64)]
            total = sum(units)
            if total:
                place = total * int(uniforms[b, k] * f32(2 ** 24)) >> 24
                run = 0
                for i, u in enumerate(units):
                    run += u
                    if run > place:
                        pick = i
                        break
                break
        out[b, 0] = count
        out[b, 1 + count] = pick
    return out


def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(f32)


@pytest.mark.parametrize("B,k,V", [(1, 1, 2), (5, 1, 100), (3, 4, 1024), (4, 7, 1025), (2, 63, 77), (2, 64, 65), (3, 70, 130), (6, 5, 32000), (1, 2, 131077)])
@pytest.mark.parametrize("certain", [False, True])
def test_verification(ctx, B, k, V, certain):
    rng = np.random.default_rng(B * 100 + k + V)
    logits = rng.standard_normal((B, k + 1, V)) * 3
    target = _softmax(logits).reshape(B * (k + 1), V)
    draft = _softmax(logits[:, :k] + rng.standard_normal((B, k, V)) * 0.4).reshape(B * k, V)
    drafted = np.array([rng.choice(V, p=r.astype(f64) / r.astype(f64).sum()) for r in draft]).reshape(B, k).astype(np.int32)
    for rep in range(4):
        u = rng.random((B, k + 1), dtype=f32)
        if rep == 1:
            u[:, :k] = 0.0     # everything that is possible is accepted
        if rep == 2:
            u[:, k] = [0.0, np.nextafter(f32(1), f32(0))][B % 2]
        if rep == 3:
            drafted[:, k // 2] = [-1, V, 2 ** 31 - 1][B % 3]  # a draft that ends early
        want = verify_reference(target, None if certain else draft, drafted, u)
        got = Tensor.from_numpy(ctx, drafted).verify_draft(Tensor.from_numpy(ctx, target), None if certain else Tensor.from_numpy(ctx, draft),
                                                           Tensor.from_numpy(ctx, u)).to_numpy()
        assert np.array_equal(got, want), rep


def test_verification_of_special_rows(ctx):
    V = 300
    p = np.zeros((8, V), f32)
    q = np.zeros((4, V), f32)
    drafted = np.array([[3], [3], [3], [3]], np.int32)
    u = np.array([[0.9, 0.5], [0.5, 0.5], [0.0, 0.999], [0.5, 2.0]], f32)
    p[0, 3], p[0, 9], q[0] = 0.25, 0.75, p[0]     # refused although nothing is left of p - q: p itself
    q[0, 3] = 1.0
    q[0, 9] = 0.8
    # sequence 1: p has no positive entry at all
    q[1, 3] = 1.0
    p[2] = np.nan
    p[4, 3], p[5, 7] = 1.0, 3.0                   # accepted; entries above 1 count as 1
    p[6, 3], p[6, 299], q[3, 3] = 0.1, 0.9, 0.9   # refused, a variate outside [0, 1)
    want = verify_reference(p, q, drafted, np.minimum(u, np.nextafter(f32(1), f32(0))))
    got = Tensor.from_numpy(ctx, drafted).verify_draft(Tensor.from_numpy(ctx, p), Tensor.from_numpy(ctx, q), Tensor.from_numpy(ctx, u)).to_numpy()
    assert np.array_equal(got, want)
    assert got[0].tolist() == [0, 9, -1] and got[1].tolist() == [0, -1, -1] and got[2].tolist() == [1, 3, 7] and got[3].tolist() == [0, 299, -1]


def test_drawn_tokens_follow_the_target(ctx):
    """Accepted and drawn tokens together are distributed as the target's own (what the method is for)."""
    rng = np.random.default_rng(8)
    V, B, reps = 6, 256, 40
    p = np.array([0.05, 0.3, 0.1, 0.25, 0.0, 0.3], f32)
    q = np.array([0.3, 0.1, 0.1, 0.1, 0.2, 0.2], f32)
    seen = np.zeros(V)
    P, Q = Tensor.from_numpy(ctx, np.tile(p, (2 * B, 1))), Tensor.from_numpy(ctx, np.tile(q, (B, 1)))
    for _ in range(reps):
        drafted = rng.choice(V, size=(B, 1), p=q.astype(f64) / q.astype(f64).sum()).astype(np.int32)
        out = Tensor.from_numpy(ctx, drafted).verify_draft(P, Q, Tensor.from_numpy(ctx, rng.random((B, 2), dtype=f32))).to_numpy()
        seen += np.bincount(out[:, 1], minlength=V)
    n = B * reps
    assert seen[4] == 0
    assert (np.abs(seen / n - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-9).all()


# -- memory and streams of other owners ---------------------------------------------------------------------------------------------------

OTHER_OWNER = """
import numpy as np, torch
torch.cuda.init()  # this process uses the HIP runtime that torch brings
from rllama_amd import Context, Tensor, TensorDType
from test_gpu_longctx import q4_decode, q4_encode
ctx = Context(0)
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(8):
        big = big @ big * 0.01  # keeps the stream busy while the calls below are queued
    x = torch.randn(64, 96, device="cuda")
    q4 = torch.zeros(64 * 96 // 32 * 20, dtype=torch.uint8, device="cuda")
    y = torch.full((64, 96), float("nan"), device="cuda")
X = Tensor.from_device(ctx, x.data_ptr(), 64, 96, TensorDType.Float32)
Q = Tensor.from_device(ctx, q4.data_ptr(), 64, 96, TensorDType.K4BitQuantization)
Y = Tensor.from_device(ctx, y.data_ptr(), 64, 96, TensorDType.Float32)
ctx.wait_stream(side.cuda_stream)
X.convert(out=Q)
Q.convert(out=Y)
ctx.release_stream(side.cuda_stream)
with torch.cuda.stream(side):
    z = y * 2
side.synchronize()
want = q4_decode(q4_encode(x.cpu().numpy()), 64, 96)
assert np.array_equal(z.cpu().numpy(), 2 * want.astype(np.float32))
for t in (X, Q, Y):
    t.free()
assert np.array_equal(y.cpu().numpy(), want.astype(np.float32))  # the memory stayed its owner's
ctx.close()
print("the same")
"""


def test_tensors_of_another_owner_on_another_stream():
    """In a process of its own: torch loads its own HIP runtime, which has to come before the library's."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    r = subprocess.run([sys.executable, "-c", OTHER_OWNER], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "the same" in r.stdout, r.stdout + r.stderr


# -- refusals ---------------------------------------------------------------------------------------------------------------------------

def refused(code, call, *args, **kw):
    with pytest.raises(RllamaHipError) as e:
        call(*args, **kw)
    assert e.value.code == code, str(e.value)


INVALID, STATE, UNSUPPORTED = 1, 5, 6


def test_refusals_of_append_and_attention(ctx):
    H, G, hd, S, n = 4, 2, 64, 16, 3
    z = lambda r, c, k="f16": Tensor.zeros(ctx, r, c, DTYPE[k])  # noqa: E731
    ck, cv, q, qkv, out = z(G * S, hd), z(G * S, hd), z(n, H * hd), z(n, (H + 2 * G) * hd), z(n, H * hd)
    fr = z(S, hd, "f32")
    i32 = Tensor.zeros(ctx, G * S, hd, TensorDType.Int32)
    ok = dict(q=q, ck=ck, cv=cv, fr=fr, H=H, G=G, S=S, at=[0])

    def append(x=qkv, q_norm=None, eps=1e-6, sinks=0, **kw):
        a = {**ok, **kw}
        x.qkv_append(a["q"], a["ck"], a["cv"], a["fr"], a["H"], a["G"], a["S"], a["at"], q_norm=q_norm, eps=eps, sinks=sinks)

    def attend(window=0, sinks=0, o=out, **kw):
        a = {**ok, **kw}
        a["q"].attn_window(a["ck"], a["cv"], a["H"], a["G"], a["S"], a["at"], window=window, sinks=sinks, out=o)

    append()
    attend()
    for f in (append, attend):
        refused(INVALID, f, H=3)                        # heads that do not share evenly
        refused(INVALID, f, G=0)
        refused(INVALID, f, S=S + 1)                    # planes of another size
        refused(INVALID, f, at=[])
        refused(INVALID, f, at=[0] * 257)
        refused(INVALID, f, at=[0, 0])                  # planes of one sequence
        refused(INVALID, f, cv=z(G * S, hd, "f32"))     # two types
        refused(INVALID, f, ck=i32, cv=i32)
        refused(INVALID, f, at=[2 ** 31 - 2])
        refused(INVALID, f, q=z(n, H * hd, "f32"))
        refused(INVALID, f, sinks=-1)
        refused(INVALID, f, sinks=S)
        refused(UNSUPPORTED, f, ck=z(G * S, 16), cv=z(G * S, 16))
        refused(STATE, f, at=[S - n + 1])               # past the table of angles; past the planes without a window
    refused(INVALID, append, q=z(n + 1, H * hd))
    refused(INVALID, append, x=z(n, H * hd))
    refused(INVALID, append, fr=z(S, 2 * hd, "f32"))
    refused(INVALID, append, fr=z(S, hd))
    refused(INVALID, append, q_norm=z(1, hd))
    refused(INVALID, append, q_norm=z(1, 2 * hd, "f32"))
    refused(INVALID, append, eps=-1.0)
    refused(INVALID, append, cv=ck)
    refused(STATE, append, x=z(15, (H + 2 * G) * hd), q=z(15, H * hd), at=[20], fr=z(64, hd, "f32"), sinks=2)  # 15 rows at once, 14 in the ring
    refused(INVALID, attend, o=q)
    refused(INVALID, attend, o=z(n, H * hd, "f32"))
    refused(INVALID, attend, window=-1)
    refused(STATE, attend, at=[40], window=12, sinks=3)  # 3 + 12 + 3 - 1 > 16
    attend(at=[40], window=11, sinks=3)
    two = z(2 * G * S, hd)
    refused(INVALID, attend, ck=two, cv=z(2 * G * S, hd), at=[0, 0])  # 3 rows for 2 sequences


def test_refusals_of_the_others(ctx):
    lib, z = ctx._lib, Tensor.zeros
    F16, F32, Q4, I32 = TensorDType.Float16, TensorDType.Float32, TensorDType.K4BitQuantization, TensorDType.Int32
    refused(INVALID, z, ctx, 4, 48, Q4)
    refused(INVALID, z, ctx, 4, 32, 4)
    a, b, q4, ids = z(ctx, 4, 64, F32), z(ctx, 4, 64, F16), z(ctx, 4, 64, Q4), z(ctx, 4, 64, I32)
    assert (q4.to_numpy() == 0).all() and ids.to_numpy().dtype == np.int32
    refused(INVALID, a.convert, out=z(ctx, 4, 32, Q4))
    refused(INVALID, z(ctx, 4, 48, F32).convert, Q4)
    refused(UNSUPPORTED, a.convert, I32)
    refused(UNSUPPORTED, ids.convert, F32)
    refused(INVALID, b.rope_table)
    refused(INVALID, a.rope_table, 0.0)
    refused(INVALID, a.softmax_rows, 1.0, out=b)
    refused(INVALID, a.softmax_rows, 1.0, out=z(ctx, 4, 65, F32))
    refused(INVALID, q4.softmax_rows)
    refused(INVALID, ids.softmax_rows)
    for t in (-1.0, float("nan"), float("inf")):
        refused(INVALID, a.softmax_rows, t)
    drafted, target, draft, u = z(ctx, 2, 3, I32), z(ctx, 8, 50, F32), z(ctx, 6, 50, F32), z(ctx, 2, 4, F32)
    drafted.verify_draft(target, draft, u)
    refused(INVALID, drafted.verify_draft, z(ctx, 6, 50, F32), draft, u)
    refused(INVALID, drafted.verify_draft, z(ctx, 8, 50, F16), draft, u)
    refused(INVALID, drafted.verify_draft, target, z(ctx, 6, 49, F32), u)
    refused(INVALID, drafted.verify_draft, target, draft, z(ctx, 2, 3, F32))
    refused(INVALID, drafted.verify_draft, target, draft, u, out=z(ctx, 2, 4, I32))
    refused(INVALID, z(ctx, 2, 3, F32).verify_draft, target, draft, u, out=z(ctx, 2, 5, I32))
    for call in (lambda: Tensor.from_device(ctx, 0, 4, 4, F32), lambda: Tensor.from_device(ctx, _pointer(a) + 4, 4, 4, F32),
                 lambda: Tensor.from_device(ctx, _pointer(a), 0, 4, F32), lambda: Tensor.from_device(ctx, _pointer(a), 1, 40, Q4)):
        refused(INVALID, call)
    # the ops that read f16 or f32 elements refuse the new types
    one = z(ctx, 1, 64, F32)
    for t in (q4, ids):
        same = z(ctx, 4, 64, t.dtype())
        refused(UNSUPPORTED, t.transpose) if t is ids else refused(INVALID, t.transpose)
        refused(UNSUPPORTED, t.hadamard_product, same)
        refused(UNSUPPORTED, t.silu)
        refused(UNSUPPORTED, t.silu_mul, same)
        refused(UNSUPPORTED, t.add, same)
        refused(INVALID, t.rmsnorm, one, 1e-6)
        refused(INVALID, t.rope_inplace, 4, 64, 0)
        refused(UNSUPPORTED, lambda: rllama_amd._lib.check(lib.rlh_matrix_mul_inplace_transposed(z(ctx, 4, 4, I32)._h, ids._h, ids._h)))
        refused(UNSUPPORTED, t.gemv, one, False, False)
        refused(INVALID, one.attn_decode, t, same, 1, 4, 1)
        refused(INVALID, t.argmax_greedy)
        buf = np.zeros(4096, np.uint8)
        refused(UNSUPPORTED if t is q4 else INVALID, lambda: rllama_amd._lib.check(lib.rlh_tensor_download(t._h, buf.ctypes.data, 65 if t is q4 else 60, None)))
