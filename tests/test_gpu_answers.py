"""The operators for many answers to one prompt against their definitions in 64 bits: tensors and products of 8 bits, attention behind a shared prefix, log
probabilities of tokens; their special rows (padding, NaN in what nobody sees, masks, ties), their refusals, and a step of them together."""
import warnings

import numpy as np
import pytest

import rllama_amd
from rllama_amd import Tensor, TensorDType
from test_gpu_longctx import DTYPE, EPS16, EPS32, INVALID, NUMPY, STATE, TYPES, UNSUPPORTED, f16, f32, f64, refused, upload, values

pytestmark = pytest.mark.gpu
F8, TILES = TensorDType.Float8, TensorDType.Float8Tiles
TINY = f32(448 * 2.0 ** -126)


# -- 8 bits -------------------------------------------------------------------------------------------------------------------------

def e4m3(t):
    """Codes of f32 values between -448 and 448: ties to even."""
    a = np.abs(t.astype(f64))
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -30))), -6) - 3)
    r = np.rint(a / step) * step  # (may reach the next power of two)
    e = np.maximum(np.floor(np.log2(np.maximum(r, 2.0 ** -30))), -6)
    code = np.where(r >= 2.0 ** -6, (e + 7) * 8 + r / np.exp2(e - 3) - 8, r * 512).astype(np.uint8)
    return code | np.signbit(t).astype(np.uint8) << 7


def decode(code):
    c = code.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8.0 + m) * np.exp2(e - 10.0), m * 2.0 ** -9)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


def encode(x, tile):
    """(codes, scales) by the definition: every step is one operation in 32 bits."""
    rows, cols = x.shape
    down = 128 if tile else 1
    codes, scales = np.zeros((rows, cols), np.uint8), np.zeros((-(-rows // down), -(-cols // 128)), f32)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * down:(i + 1) * down, j * 128:(j + 1) * 128]
            v = x[at].astype(f32)
            if not np.isfinite(v).all():
                scales[i, j] = np.nan
                continue
            a = max(np.abs(v).max(), TINY)
            scales[i, j] = a / f32(448)
            codes[at] = e4m3(np.clip(v * (f32(448) * (f32(1) / a)), f32(-448), f32(448)))
    return codes, scales


def stands_for(codes, scales, tile):
    s = scales.astype(f64).repeat(128 if tile else 1, 0)[:codes.shape[0]].repeat(128, 1)[:, :codes.shape[1]]
    return decode(codes) * s


def parts(t):
    """(codes, scales) of a tensor of 8 bits."""
    b, count = t.to_numpy(), t.rows() * t.cols()
    return b[:count].reshape(t.rows(), t.cols()), b[count:].view(f32).reshape(-1, -(-t.cols() // 128))


@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (3, 144), (37, 400), (128, 128), (129, 272), (300, 1008)])
@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("tile", [False, True])
def test_conversion_to_and_from_8_bits_is_its_definition(ctx, rows, cols, kind, tile):
    rng = np.random.default_rng(rows + cols)
    with np.errstate(over="ignore"):
        x = (rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-9, 6, (rows, 1)))).astype(NUMPY[kind])
    if rows > 30:
        x[0, 3] = np.nan
        x[min(rows - 1, 140), cols - 1] = np.inf
        x[2, :128] = 0.0
        x[3, :128] = 0.37
        x[4, :128] = np.linspace(-448, 448, 128)
        x[4, 5:12] = [17, 19, 21, 23, 2.0 ** -9, 3 * 2.0 ** -10, 2.0 ** -10]  # ties, and the smallest numbers
        if kind == "f32":
            x[5, :128] *= f32(1e-40)
            x[6, :128] = 3e38
    t = Tensor.from_numpy(ctx, x).convert(TILES if tile else F8)
    codes, scales = encode(x, tile)
    got_codes, got_scales = parts(t)
    assert np.array_equal(got_scales, scales, equal_nan=True)
    assert np.array_equal(got_codes, codes)
    want = stands_for(codes, scales, tile).astype(f32)  # (24 bits hold a product of 4 and 24 rounded once)
    back = t.convert(TensorDType.Float32).to_numpy()
    assert np.array_equal(back, want, equal_nan=True)
    with np.errstate(over="ignore"):
        assert np.array_equal(t.convert(TensorDType.Float16).to_numpy(), want.astype(f16), equal_nan=True)
    again = Tensor.from_f8(ctx, codes, scales)
    assert again.dtype() == (TILES if tile and rows > 1 else F8)
    assert np.array_equal(t.clone().to_numpy(), again.to_numpy()) or np.isnan(scales).any()


def test_every_code_of_8_bits(ctx):
    codes = np.arange(256, dtype=np.uint8).reshape(2, 128)
    t = Tensor.from_f8(ctx, codes, np.array([[1.0], [0.37]], f32))
    want = (decode(codes) * np.array([[1.0], [f64(f32(0.37))]])).astype(f32)
    assert np.array_equal(t.convert(TensorDType.Float32).to_numpy(), want, equal_nan=True)


PRODUCTS = [
    # rows, results, depth
    (1, 1, 16), (1, 5, 128), (1, 129, 144), (1, 4096, 4096), (2, 300, 2064), (5, 17, 1008), (7, 1000, 11008), (16, 128, 128), (16, 515, 640), (17, 256, 1024), (31, 33, 4112),
    (33, 700, 400), (64, 640, 2816), (65, 257, 1296), (96, 96, 96), (100, 1111, 528), (128, 256, 256), (129, 130, 272), (131, 1024, 2816), (256, 256, 1024), (257, 511, 384),
    (300, 2000, 1040), (513, 384, 5120), (1024, 1024, 512), (40, 4099, 304),
]


def product_bound(x, w, k, kind):
    """What a sum may be off by.  A block's 128 products are exact in f32 (8 bits) and added up in f32, the blocks' sums times their scales as well: an addition each, and
    two roundings per block.  For f16 results the matrix instruction for 8 bits may be used, which adds up eight products at a time and leaves out what each has below
    2^-13 of the largest's power of two: seven such parts of a group at most."""
    size = np.abs(x) @ np.abs(w).T
    off = size * EPS32 * (4 + np.sqrt(128) + np.sqrt(-(-k // 128)))
    if kind == "f16":
        group = lambda a: np.abs(a).reshape(len(a), k // 8, 8).max(-1)  # noqa: E731
        off = off + 7 * 2.0 ** -13 * (group(x) @ group(w).T)
    return off


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("source,result", [("f16", "f16"), ("f32", "f32"), ("f8", "f16"), ("f8", "f32")])
def test_product(ctx, m, n, k, source, result):
    rng = np.random.default_rng(m * 3 + n * 5 + k)
    x = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal((1, k)))).astype(f32 if source == "f8" else NUMPY[source])
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(f32)
    W = Tensor.from_numpy(ctx, w).convert(TILES)
    X = Tensor.from_numpy(ctx, x)
    wide = stands_for(*parts(W), True)
    eight = X.convert(F8)
    x8 = stands_for(*parts(eight), False)
    out = Tensor.from_numpy(ctx, np.full((m, n), np.nan, NUMPY[result]))
    (eight if source == "f8" else X).matrix_mul_f8(W, out=out)
    got = out.to_numpy().astype(f64)
    want = x8 @ wide.T
    tol = product_bound(x8, wide, k, result) + (EPS16 * np.abs(want) + 2.0 ** -25 if result == "f16" else EPS32 * np.abs(want))
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    again = (eight if source == "f8" else X).matrix_mul_f8(W, dtype=DTYPE[result])
    assert np.array_equal(again.to_numpy(), out.to_numpy())


@pytest.mark.parametrize("m,n,k", [(1, 200, 384), (20, 300, 272), (70, 300, 272), (200, 300, 400)])
def test_product_of_values_that_are_not_finite(ctx, m, n, k):
    """They reach the rows and columns that they belong to, and no others; zeros, and scales of every size."""
    rng = np.random.default_rng(m)
    x, w = rng.standard_normal((m, k)).astype(f32), rng.standard_normal((n, k)).astype(f32)
    if m > 1:
        x[m // 2, 5] = np.inf
        x[0] = 0.0
    x[-1] *= f32(1e30)
    w[260 if n > 260 else 130, 140] = np.nan  # the whole tile
    lost = np.s_[256:] if n > 260 else np.s_[128:]
    got = Tensor.from_numpy(ctx, x).matrix_mul_f8(Tensor.from_numpy(ctx, w).convert(TILES)).to_numpy()
    nan = np.zeros((m, n), bool)
    nan[:, lost] = True
    if m > 1:
        nan[m // 2] = True
    assert np.array_equal(np.isnan(got), nan)
    if m > 1:
        assert (got[0][~nan[0]] == 0).all()
    assert (np.abs(got[-1][~nan[-1]]) > 1e25).any()


# -- attention behind a shared prefix ---------------------------------------------------------------------------------------------------

SHARED = [
    # hd, heads, kv heads, rows of a text, prefix, its planes' rows, the texts' rows, positions of the first rows
    (128, 4, 4, 1, 1, 1, 3, [0]),
    (128, 4, 4, 1, 0, 0, 40, [37, 0, 5]),                    # no prefix
    (64, 2, 2, 1, 33, 40, 300, [255, 16, 31, 32, 0, -1]),    # an idle slot
    (32, 8, 2, 1, 1000, 1000, 70, [64, 3, 0]),
    (128, 16, 1, 1, 2055, 2060, 100, [99, 2]),
    (128, 34, 2, 1, 333, 400, 60, [50, 8]),                  # 17 heads share a key head
    (128, 8, 1, 5, 777, 777, 90, [70, 80, 1]),
    (64, 7, 7, 3, 150, 171, 160, [100, -2, -3, 0]),          # padding in front
    (64, 4, 2, 33, 95, 95, 64, [0, 20]),
    (128, 2, 1, 130, 300, 300, 200, [0, 57, -40]),
    (32, 3, 3, 71, 31, 64, 400, [300, 0]),
    (128, 8, 8, 1, 5000, 5100, 20, [3] * 20),
    (128, 32, 8, 1, 700, 700, 40, list(range(33)) + [-1]),
    (64, 16, 2, 2, 1300, 1300, 500, [490, 0, 17, 200, 3, 333, 64, 65, 31, 32]),
    (128, 4, 2, 9, 129, 129, 700, [600, 690, 0]),
    (32, 12, 4, 1, 9000, 9000, 8, [7] * 64),
    (128, 16, 2, 1, 30, 30, 3000, [2990, 1, 1500]),          # own texts much longer than the prefix
    (128, 5, 1, 60, 2107, 2107, 64, [0] * 6),
    (64, 1, 1, 1, 64, 64, 64, [63] * 256),
    (64, 6, 2, 11, 200, 210, 150, [130, 0, -3, 64, 7, -11, 100, 139, 1, 55]),  # up to five texts in a block of 128 rows
    (128, 4, 1, 10, 0, 0, 300, [290, 0, 100, -5, 17, 200]),
    (128, 10, 2, 61, 700, 700, 61, [0] * 6),
]


def shared_reference(q, PK, PV, K, V, starts):
    """q [B, n, H, hd], prefix planes [G, P, hd], own planes [B, G, S, hd] in 64 bits; also the bound of the error that f32 arithmetic may leave."""
    B, n, H, hd = q.shape
    G = PK.shape[0]
    out, bound = np.zeros(q.shape), np.zeros((B, n, H, 1))
    for b, start in enumerate(starts):
        for i in range(n):
            p = start + i
            if p < 0:
                continue
            for g in range(G):
                k, v = np.concatenate([PK[g], K[b, g, :p + 1]]), np.concatenate([PV[g], V[b, g, :p + 1]])
                hs = slice(g * (H // G), (g + 1) * (H // G))
                s = q[b, i, hs] @ k.T / np.sqrt(hd)
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[b, i, hs] = w @ v
                # a score is off by some roundings of a sum of hd terms, each weight by as much, the sums over the positions by theirs
                size = (np.abs(q[b, i, hs]) @ np.abs(k).T).max(-1, keepdims=True) / np.sqrt(hd)
                bound[b, i, hs] = np.abs(v).max() * (8 * np.sqrt(hd) * EPS32 * size + (4 * np.sqrt(len(k)) + 16) * EPS32)
    return out, bound


def shared_case(ctx, hd, H, G, n, P, rows, S, starts, kind, cache, spread=1.5, seed=0):
    """A call on random planes, NaN in everything that no row sees: (result, definition, bound, arguments)."""
    rng = np.random.default_rng(hd * 31 + H * 7 + n + P + S + seed)
    B = len(starts)
    q = (rng.standard_normal((B, n, H, hd)) * spread).astype(NUMPY[kind])
    PK, PV = (rng.standard_normal((G, max(1, rows), hd)) for _ in range(2))
    K, V = (rng.standard_normal((B, G, S, hd)) for _ in range(2))
    for x in (PK, PV):
        x[:, P:] = np.nan
    for x in (K, V):
        for b, start in enumerate(starts):
            x[b, :, max(0, start + n):] = np.nan
    pk, pv, ck, cv = (upload(ctx, x.reshape(-1, hd), cache) for x in (PK, PV, K, V))
    PK, PV = (values(t).reshape(G, -1, hd)[:, :P] for t in (pk, pv))
    K, V = (values(t).reshape(B, G, S, hd) for t in (ck, cv))
    want, bound = shared_reference(q.astype(f64), PK, PV, K, V, starts)
    Q = Tensor.from_numpy(ctx, q.reshape(B * n, H * hd))
    out = Tensor.from_numpy(ctx, np.full((B * n, H * hd), np.nan, NUMPY[kind]))
    args = (pk if rows else None, pv if rows else None, P, ck, cv, H, G, S, starts)
    Q.attn_shared(*args, out=out)
    tops = [np.nanmax(np.abs(x)) for x in (PV, V) if x.size]
    if kind == "f16":  # the result is rounded to f16; the weights may be
        bound = bound + 2 * EPS16 * max(tops)
    return out.to_numpy(), want, bound, Q, args


@pytest.mark.parametrize("hd,H,G,n,P,rows,S,starts", SHARED)
@pytest.mark.parametrize("kind,cache", TYPES)
def test_attention_behind_a_shared_prefix(ctx, hd, H, G, n, P, rows, S, starts, kind, cache):
    out, want, bound, Q, args = shared_case(ctx, hd, H, G, n, P, rows, S, starts, kind, cache)
    got = out.astype(f64).reshape(want.shape)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / np.maximum(bound, 1e-30)
    assert worst.max() <= 1, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))
    for b, start in enumerate(starts):
        assert (got[b, :max(0, min(n, -start))] == 0).all()
    # the same again: no sum depends on which workgroup came first
    assert np.array_equal(Q.attn_shared(*args).to_numpy(), out)


@pytest.mark.parametrize("kind,cache", TYPES)
@pytest.mark.parametrize("hd,n,P,starts", [(32, 40, 256, [-40, -40, -99]), (32, 2, 256, [-2, -9]), (64, 1, 0, [-2] * 40), (128, 50, 0, [-50]), (128, 1, 500, [-1] * 40), (64, 1, 0, [-1])])
def test_nothing_but_padding(ctx, kind, cache, hd, n, P, starts):
    with np.errstate(all="ignore"), warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (no position is seen, and all of them are NaN)
        out = shared_case(ctx, hd, 4, 4, n, P, P, 40, starts, kind, cache)[0]
    assert (out == 0).all()


@pytest.mark.parametrize("P", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1023, 1025, 3000])
@pytest.mark.parametrize("kind,cache,B", [("f16", "f16", 1), ("f16", "f16", 20), ("f16", "q4", 5), ("f32", "f32", 3)])
def test_prefixes_of_every_length(ctx, P, kind, cache, B):
    out, want, bound, _, _ = shared_case(ctx, 128, 4, 2, 1, P, P + 3, 70, [(7 * b) % 64 for b in range(B)], kind, cache, seed=P)
    assert (np.abs(out.astype(f64).reshape(want.shape) - want) <= bound).all()


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("n,B", [(1, 3), (1, 40), (20, 5), (70, 4)])
def test_scores_far_apart(ctx, kind, n, B):
    """Scores of several hundred, rising and falling along prefix and text: the running maximum moves all the time, weights underflow, and one of the two parts may hold all of it."""
    rng = np.random.default_rng(9)
    H, hd, P, S = 2, 64, 300, 200
    for order in (1, -1, 0):
        ramp = np.linspace(-40, 40, P + S) * order if order else rng.permutation(np.linspace(-40, 40, P + S))
        K = rng.standard_normal((B, H, P + S, hd)) * 0.1
        K[..., 0] = ramp
        K[:, :, :P] = K[:1, :, :P]
        V = rng.standard_normal((B, H, P + S, hd))
        V[:, :, :P] = V[:1, :, :P]
        q = rng.standard_normal((B, n, H, hd))
        q[..., 0] = 60.0  # scores from -300 to 300
        q, K, V = (x.astype(NUMPY[kind]).astype(f64) for x in (q, K, V))
        starts = [(S - n) * (b + 1) // B for b in range(B)]
        planes = [K[0, :, :P], V[0, :, :P], K[:, :, P:], V[:, :, P:]]
        want, bound = shared_reference(q, *planes, starts)
        pk, pv, ck, cv = (upload(ctx, np.ascontiguousarray(x).reshape(-1, hd), kind) for x in planes)
        got = Tensor.from_numpy(ctx, q.reshape(B * n, -1).astype(NUMPY[kind])).attn_shared(pk, pv, P, ck, cv, H, H, S, starts).to_numpy().astype(f64).reshape(want.shape)
        # near the top a score of 300 has a unit of 2^-15 in f32: exp's argument is off by as much whatever the operands' type
        tol = bound + 2 * np.abs(V).max() * 300 * 4 * EPS32 + (2 * EPS16 * np.abs(V).max() if kind == "f16" else 0)
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4"), ("f32", "f32"), ("f32", "q4")])
@pytest.mark.parametrize("B,n,group", [(3, 1, 2), (30, 1, 4), (4, 20, 1), (12, 7, 3), (5, 20, 2), (3, 34, 4)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(ctx, kind, cache, B, n, group, value):
    G, hd, P, S = 2, 32, 150, 64
    rng = np.random.default_rng(B)
    starts = [30] * B
    q = rng.standard_normal((B, n, G * group, hd)).astype(NUMPY[kind])
    for where in ("prefix", "text"):
        PK, PV = (rng.standard_normal((G, P, hd)) for _ in range(2))
        K, V = (rng.standard_normal((B, G, S, hd)) for _ in range(2))
        if where == "prefix":
            PV[1, 70, 5] = value
        else:
            V[1, 1, 30 + n // 2, 5] = value  # seen from the middle row of the second text on
        pk, pv, ck, cv = (upload(ctx, x.reshape(-1, hd), cache) for x in (PK, PV, K, V))
        got = Tensor.from_numpy(ctx, q.reshape(B * n, -1)).attn_shared(pk, pv, P, ck, cv, G * group, G, S, starts).to_numpy().reshape(B, n, G, group, hd)
        hit = np.zeros(got.shape, bool)
        rows = np.s_[:, :, 1] if where == "prefix" else np.s_[1, n // 2:, 1]
        if cache == "q4":
            hit[rows] = True  # (of 4 bits the whole group is NaN)
        else:
            hit[rows + (Ellipsis, 5)] = True
        want = np.nan if cache == "q4" or np.isnan(value) else np.inf
        assert np.array_equal(got[hit], np.full(hit.sum(), want), equal_nan=True) and np.isfinite(got[~hit]).all()


def test_keys_that_are_not_finite(ctx):
    """A key of -infinity scores has no weight; a NaN in it spoils the rows that see it and no others."""
    G, hd, P, S, B = 1, 64, 100, 40, 3
    rng = np.random.default_rng(4)
    q = np.abs(rng.standard_normal((B, hd))).astype(f32)
    PK, PV, K, V = rng.standard_normal((P, hd)), rng.standard_normal((P, hd)), rng.standard_normal((B * S, hd)), rng.standard_normal((B * S, hd))
    PK[50] = -np.inf
    K[S + 10, 3] = np.nan
    starts = [20, 20, 5]
    for kind in ("f16", "f32"):
        t = [upload(ctx, x, kind) for x in (PK, PV, K, V)]
        Q = Tensor.from_numpy(ctx, q.astype(NUMPY[kind]))
        got = Q.attn_shared(t[0], t[1], P, t[2], t[3], 1, G, S, starts).to_numpy()
        assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()
        keep = np.arange(P) != 50
        pk, pv = (upload(ctx, x[keep], kind) for x in (PK, PV))
        other = Q.attn_shared(pk, pv, P - 1, t[2], t[3], 1, G, S, starts).to_numpy()
        assert np.abs(got[[0, 2]].astype(f64) - other[[0, 2]]).max() <= (2 * EPS16 if kind == "f16" else 64 * EPS32) * np.abs(PV).max()
    # nothing but keys of -infinity: zeros
    dead = upload(ctx, np.full((P, hd), -np.inf), "f32"), upload(ctx, np.full((B * S, hd), -np.inf), "f32")
    got = Tensor.from_numpy(ctx, q).attn_shared(dead[0], upload(ctx, PV, "f32"), P, dead[1], upload(ctx, V, "f32"), 1, G, S, starts).to_numpy()
    assert (got == 0).all()


def test_the_same_as_attention_over_whole_texts(ctx):
    """A prefix copied in front of every text gives what the shared one does, up to the results' rounding."""
    H, G, hd, P, S, B = 8, 2, 64, 130, 40, 5
    rng = np.random.default_rng(6)
    PK, PV, K, V = (rng.standard_normal((r, hd)).astype(f16) for r in (G * P, G * P, B * G * S, B * G * S))
    starts = [0, 39, 7, 20, 31]
    q = Tensor.from_numpy(ctx, rng.standard_normal((B, H * hd)).astype(f16))
    shared = q.attn_shared(*(Tensor.from_numpy(ctx, x) for x in (PK, PV)), P, *(Tensor.from_numpy(ctx, x) for x in (K, V)), H, G, S, starts).to_numpy()
    whole = [np.concatenate([np.broadcast_to(p.reshape(1, G, P, hd), (B, G, P, hd)), x.reshape(B, G, S, hd)], 2).reshape(-1, hd) for p, x in ((PK, K), (PV, V))]
    apart = q.attn_window(*(Tensor.from_numpy(ctx, x) for x in whole), H, G, P + S, [P + s for s in starts]).to_numpy()
    assert np.abs(shared.astype(f64) - apart).max() <= 2 * EPS16 * np.abs(PV.astype(f64)).max()


@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4"), ("f32", "f32")])
def test_a_large_batch_is_its_texts(ctx, kind, cache):
    """More blocks of rows than there is room for at a time, of which the last ones are cut: the same as every text by itself, which is cut into pieces.  Both are within
    the bound of the results of each other."""
    H, hd, n, B, P, S = 32, 64, 66, 20, 3000, 70
    rng = np.random.default_rng(20)
    pk, pv = (upload(ctx, rng.standard_normal((H * P, hd)), cache) for _ in range(2))
    own = [rng.standard_normal((B, H * S, hd)) for _ in range(2)]
    starts = [b % 7 - 3 for b in range(B)]
    q = rng.standard_normal((B, n, H * hd)).astype(NUMPY[kind])
    got = Tensor.from_numpy(ctx, q.reshape(B * n, -1)).attn_shared(pk, pv, P, *(upload(ctx, x.reshape(-1, hd), cache) for x in own), H, H, S, starts).to_numpy().reshape(B, n, -1).astype(f64)
    for b in range(B):
        alone = Tensor.from_numpy(ctx, q[b]).attn_shared(pk, pv, P, *(upload(ctx, x[b], cache) for x in own), H, H, S, starts[b:b + 1]).to_numpy().astype(f64)
        size = max(np.abs(x).max() for x in own + [values(pv)])
        scores = np.abs(q[b].astype(f64)).max() * hd ** 0.5 * size  # (no score is larger)
        bound = size * (8 * np.sqrt(hd) * EPS32 * scores + (4 * np.sqrt(P + S) + 16) * EPS32) + (2 * EPS16 * size if kind == "f16" else 0)
        assert (np.abs(got[b] - alone) <= 2 * bound).all()


# -- log probabilities --------------------------------------------------------------------------------------------------------------------

def logprobs_reference(x, temperature):
    z = x.astype(f64) / f64(f32(temperature))
    top = z.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        z = z - top
        e = np.exp(z)
        s = e.sum(-1, keepdims=True)
        p = z - np.log(s)
        h = np.log(s) - np.where(e > 0, e * z, 0).sum(-1, keepdims=True) / s
    return p, h


def first_of_the_largest(x, k):
    return np.argsort(-x.astype(f64), axis=-1, kind="stable")[:, :k].astype(np.int32)


@pytest.mark.parametrize("vocab", [1, 3, 33, 63, 64, 65, 1000, 1023, 2049, 4097, 8193, 32000, 32001, 50257, 131075])
@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("temperature,top,m", [(1.0, 20, 1), (0.3, 5, 3), (1.7, 0, 1), (0.8, 32, 70), (1.0, 1, 0)])
def test_logprobs(ctx, vocab, kind, temperature, top, m):
    rng = np.random.default_rng(vocab + top)
    rows = 5
    x = (rng.standard_normal((rows, vocab)) * np.array([[0.01], [1], [4], [4], [30]])).astype(NUMPY[kind])
    if vocab > 2:
        x[2, ::2] = -np.inf
        x[3] = np.round(x[3])  # many equal ones
    top = min(top, vocab)
    tokens = rng.integers(0, vocab, (rows, m)).astype(np.int32) if m else None
    if m > 1:
        tokens[:, 0] = -1
        tokens[:, 1] = [-7, vocab, 2 ** 31 - 1, 0, vocab - 1]
    got = Tensor.from_numpy(ctx, x).token_logprobs(Tensor.from_numpy(ctx, tokens) if m else None, temperature, top)
    want, entropy = logprobs_reference(x, temperature)
    # off by the rounding of z (one of the difference, one of 1 / temperature, one of the product), of the logarithm, and of the sum, whose terms are all positive
    finite = np.where(np.isfinite(x), x.astype(f64), 0)
    tol = EPS32 * (8 + 2 * np.sqrt(vocab) + 6 * np.abs(want) + 6 * np.abs(np.log(vocab)))
    if m:
        inside = (tokens >= 0) & (tokens < vocab)
        at = np.where(inside, tokens, 0)
        w = np.where(inside, np.take_along_axis(want, at, 1), np.where(tokens < 0, 0.0, -np.inf))
        g, t = got[0].to_numpy().astype(f64), np.take_along_axis(tol, at, 1)
        same = np.isneginf(w) & np.isneginf(g)
        assert (same | (np.abs(np.where(same, 0, g) - np.where(same, 0, w)) <= t)).all()
    g = got[1].to_numpy().astype(f64)
    # the entropy's sum over terms p log p, each off by its exponent's roundings; near zero it is as exact as its terms are
    assert (np.abs(g - entropy) <= EPS32 * (16 + 2 * np.sqrt(vocab)) * (np.abs(entropy) + np.log(vocab) * (vocab > 1) * 8)).all()
    if top:
        ids = first_of_the_largest(x, top)
        assert np.array_equal(got[2].to_numpy(), ids)
        w, g, t = (np.take_along_axis(a, ids, 1) for a in (want, want, tol))
        g = got[3].to_numpy().astype(f64)
        same = np.isneginf(w) & np.isneginf(g)
        assert (same | (np.abs(np.where(same, 0, g) - np.where(same, 0, w)) <= t)).all()


def test_logprobs_near_certainty(ctx):
    """One token far ahead of the others: its log probability, and the entropy, are as exact as the others' weights, not as 1 minus them."""
    x = np.zeros((6, 3001), f32)
    for r, ahead in enumerate((5, 20, 30, 40, 60, 80)):
        x[r, 17 * r] = ahead
    t = Tensor.from_numpy(ctx, np.array([[17 * r] for r in range(6)], np.int32))
    got = Tensor.from_numpy(ctx, x).token_logprobs(t, 1.0, 2)
    rest = 3000 * np.exp(-np.array([5, 20, 30, 40, 60, 80], f64))
    entropy = np.log1p(rest) + rest / (1 + rest) * np.array([5, 20, 30, 40, 60, 80])
    assert np.allclose(got[0].to_numpy()[:, 0], -np.log1p(rest), rtol=2e-5, atol=0)  # (an exponent of 80 has a unit of 2^-17: exp is off by 7e-6 of itself)
    assert np.allclose(got[1].to_numpy()[:, 0], entropy, rtol=2e-5, atol=0)
    assert np.array_equal(got[2].to_numpy()[:, 0], [17 * r for r in range(6)]) and np.array_equal(got[2].to_numpy()[:, 1], [1, 0, 0, 0, 0, 0])


@pytest.mark.parametrize("vocab", [700, 5000, 32000, 40000])
@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_logprobs_of_special_rows(ctx, vocab, kind):
    low, high = np.finfo(NUMPY[kind]).min, np.finfo(NUMPY[kind]).max
    x = np.zeros((9, vocab), NUMPY[kind])
    x[0] = -np.inf
    x[1, 5] = np.nan
    x[2, vocab - 1] = np.inf
    x[3] = -np.inf
    x[3, [13, 400]] = low           # masks of the type's lowest value among masks of -infinity
    x[4] = high
    x[5, [7, 9, 600]] = 2.0
    x[6] = low
    x[7, ::2] = -0.0                # equal to the others
    x[8, :] = low
    x[8, [3, 699]] = [1.0, 2.0]     # all but two masked
    tokens = np.tile(np.array([[13, -1, vocab, 0]], np.int32), (9, 1))
    g = [t.to_numpy() for t in Tensor.from_numpy(ctx, x).token_logprobs(Tensor.from_numpy(ctx, tokens), 0.5, 32)]
    logv = np.log(vocab)
    assert (g[0][0] == [-np.inf, 0, -np.inf, -np.inf]).all() and g[1][0] == 0 and np.array_equal(g[2][0], np.arange(32)) and (g[3][0] == -np.inf).all()
    for r in (1, 2):
        assert np.array_equal(np.isnan(g[0][r]), [True, False, True, True]) and g[0][r, 1] == 0 and np.isnan(g[1][r]) and (g[2][r] == -1).all() and np.isnan(g[3][r]).all()
    assert np.allclose(g[0][3], [-np.log(2), 0, -np.inf, -np.inf]) and np.isclose(g[1][3], np.log(2)) and np.array_equal(g[2][3], [13, 400] + [i for i in range(31) if i != 13])
    for r in (4, 6, 7):
        assert np.allclose(g[0][r], [-logv, 0, -np.inf, -logv], rtol=1e-6) and np.allclose(g[1][r], logv, rtol=1e-6) and np.array_equal(g[2][r], np.arange(32))
        assert np.allclose(g[3][r], -logv, rtol=1e-6)
    assert np.array_equal(g[2][5], [7, 9, 600] + [i for i in range(31) if i not in (7, 9)])
    assert np.array_equal(g[2][8][:2], [699, 3]) and np.allclose(g[3][8][:2], -np.log1p(np.exp([-2.0, 2.0])), rtol=1e-6)
    assert np.array_equal(g[2][8][2:], [i for i in range(31) if i != 3])


@pytest.mark.parametrize("vocab", [600, 5000, 32000, 40000])
@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("larger", [3, 27, 101, 203, 255, 256, 257, 450])
def test_logprobs_of_larger_ones_side_by_side(ctx, vocab, kind, larger):
    """The larger entries lie together, at the front, in the middle and at the end, and all others are equal: what bounds the most probable ones from below is met by all."""
    rng = np.random.default_rng(larger)
    x = np.zeros((12, vocab), NUMPY[kind])
    for r in range(12):
        at = [0, (vocab - larger) // 2 + r, vocab - larger][r % 3]
        x[r, at:at + larger] = rng.permutation(larger) / 64 + 0.5
        if r >= 6:
            x[r, x[r] == 0] = -np.inf
    g = [t.to_numpy() for t in Tensor.from_numpy(ctx, x).token_logprobs(None, 0.9, 32)[2:]]
    ids = first_of_the_largest(x, 32)
    assert np.array_equal(g[0], ids)
    want = np.take_along_axis(logprobs_reference(x, 0.9)[0], ids, 1)
    with np.errstate(invalid="ignore"):
        assert ((g[1] == want) | (np.abs(g[1] - want) <= EPS32 * (8 + 2 * np.sqrt(vocab) + 6 * np.abs(want) + 6 * np.log(vocab)))).all()


# -- refusals ---------------------------------------------------------------------------------------------------------------------------

def test_refusals_of_the_attention(ctx):
    H, G, hd, S, n, P = 4, 2, 64, 16, 3, 20
    z = lambda r, c, k="f16": Tensor.zeros(ctx, r, c, DTYPE[k])  # noqa: E731
    ok = dict(q=z(n, H * hd), pk=z(G * P, hd), pv=z(G * P, hd), P=P, ck=z(G * S, hd), cv=z(G * S, hd), H=H, G=G, S=S, at=[0], out=z(n, H * hd))

    def call(**kw):
        a = {**ok, **kw}
        a["q"].attn_shared(a["pk"], a["pv"], a["P"], a["ck"], a["cv"], a["H"], a["G"], a["S"], a["at"], out=a["out"])

    call()
    call(P=0)
    call(P=0, pk=None, pv=None)
    call(at=[-3])
    refused(INVALID, call, H=3)
    refused(INVALID, call, G=0)
    refused(INVALID, call, S=S + 1)
    refused(INVALID, call, at=[])
    refused(INVALID, call, at=[0] * 257)
    refused(INVALID, call, at=[0, 0])
    refused(INVALID, call, P=P + 1)
    refused(INVALID, call, P=-1)
    refused(INVALID, call, pk=None, pv=None)
    refused(INVALID, call, pv=None)
    refused(INVALID, call, pv=None, P=0)
    refused(INVALID, call, cv=z(G * S, hd, "f32"))
    refused(INVALID, call, pk=z(G * P, hd, "f32"), pv=z(G * P, hd, "f32"))
    refused(INVALID, call, pk=z(G * P, 2 * hd), pv=z(G * P, 2 * hd))
    refused(INVALID, call, pk=z(G * P + 1, hd), pv=z(G * P + 1, hd))
    for kind in (TensorDType.Int32, F8):
        t = Tensor.zeros(ctx, G * S, hd, kind)
        refused(INVALID, call, ck=t, cv=t)
        refused(INVALID, call, q=Tensor.zeros(ctx, n, H * hd, kind))
    refused(INVALID, call, q=z(n, H * hd, "f32"))
    refused(INVALID, call, q=z(n, hd))
    refused(INVALID, call, out=ok["q"])
    refused(INVALID, call, out=z(n + 1, H * hd))
    refused(UNSUPPORTED, call, ck=z(G * S, 16), cv=z(G * S, 16))
    refused(STATE, call, at=[S - n + 1])
    refused(STATE, call, at=[2 ** 31 - 1])
    two = z(2 * G * S, hd)
    refused(INVALID, call, ck=two, cv=two, at=[0, 0])  # 3 rows for 2 texts


def test_refusals_of_the_others(ctx):
    z = lambda r, c, k: Tensor.zeros(ctx, r, c, k)  # noqa: E731
    F16, F32, I32, Q4 = TensorDType.Float16, TensorDType.Float32, TensorDType.Int32, TensorDType.K4BitQuantization
    # tensors of 8 bits
    for kind in (F8, TILES):
        refused(INVALID, z, 4, 24, kind)
        refused(INVALID, lambda: Tensor.from_device(ctx, 4096, 4, 24, kind))
        t = z(4, 64, kind)
        assert (t.to_numpy() == 0).all()
        refused(UNSUPPORTED, t.convert, Q4)
        refused(UNSUPPORTED, z(4, 64, Q4).convert, kind)
        refused(UNSUPPORTED, t.convert, F8 if kind == TILES else TILES)
        refused(UNSUPPORTED, t.convert, I32)
        refused(UNSUPPORTED, t.silu)
        refused(UNSUPPORTED, t.hadamard_product, z(4, 64, kind))
        refused(INVALID, t.transpose)
        refused(UNSUPPORTED, t.matrix_mul_transposed, z(16, 64, kind))
        refused(INVALID, t.softmax_rows)
        buf = np.zeros(4096, np.uint8)
        refused(UNSUPPORTED, lambda: rllama_amd._lib.check(ctx._lib.rlh_tensor_download(t._h, buf.ctypes.data, 65, None)))
    # products
    x, w = z(3, 64, F16), z(32, 64, TILES)
    x.matrix_mul_f8(w)
    refused(INVALID, x.matrix_mul_f8, z(32, 64, F8))
    refused(INVALID, x.matrix_mul_f8, z(32, 64, F16))
    refused(INVALID, x.matrix_mul_f8, z(32, 80, TILES))
    refused(INVALID, x.matrix_mul_f8, w, out=z(3, 33, F16))
    refused(INVALID, x.matrix_mul_f8, w, out=z(4, 32, F16))
    refused(INVALID, x.matrix_mul_f8, w, out=z(3, 32, I32))
    refused(INVALID, z(3, 64, Q4).matrix_mul_f8, w, out=z(3, 32, F16))
    refused(INVALID, z(3, 64, TILES).matrix_mul_f8, w, out=z(3, 32, F16))
    square = z(32, 32, F16)
    refused(INVALID, square.matrix_mul_f8, z(32, 32, TILES), out=square)
    # log probabilities
    logits, tokens = z(3, 50, F32), z(3, 2, I32)
    logits.token_logprobs(tokens, 1.0, 5)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-31, 1e31):
        refused(INVALID, logits.token_logprobs, tokens, t)
    refused(INVALID, tokens.token_logprobs)
    refused(INVALID, logits.token_logprobs, z(4, 2, I32), logprobs=z(4, 2, F32))
    refused(INVALID, logits.token_logprobs, z(3, 2, F32))
    refused(INVALID, logits.token_logprobs, tokens, logprobs=z(3, 1, F32))
    refused(INVALID, logits.token_logprobs, tokens, logprobs=z(3, 2, F16))
    refused(INVALID, logits.token_logprobs, tokens, entropy=z(3, 2, F32))
    refused(INVALID, logits.token_logprobs, tokens, entropy=z(3, 1, F16))
    refused(INVALID, logits.token_logprobs, tokens, 1.0, 5, top_logprobs=z(3, 6, F32))
    refused(INVALID, logits.token_logprobs, top_ids=z(3, 5, F32))
    refused(INVALID, z(3, 8, F32).token_logprobs, tokens, 1.0, 9)
    refused(UNSUPPORTED, logits.token_logprobs, tokens, 1.0, 33)
    lib = ctx._lib
    refused(INVALID, lambda: rllama_amd._lib.check(lib.rlh_token_logprobs(None, None, None, None, logits._h, None, 1.0)))
    refused(INVALID, lambda: rllama_amd._lib.check(lib.rlh_token_logprobs(None, None, None, None, logits._h, tokens._h, 1.0)))
    # angles
    table = z(4, 64, F32)
    refused(INVALID, table.rope_table_from, -1)
    refused(INVALID, table.rope_table_from, 2 ** 31 - 3)
    refused(INVALID, table.rope_table_from, 5, 0.0)
    refused(INVALID, z(4, 64, F16).rope_table_from, 5)
    whole = z(104, 64, F32).rope_table().to_numpy()
    assert np.array_equal(table.rope_table_from(100).to_numpy(), whole[100:])


# -- together -----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", ["f16", "q4", "f32"])
def test_a_step_of_many_answers(ctx, cache):
    """A prompt of 150 positions read once, then three steps of seven answers of different lengths: product of 8 bits, append behind the prefix, attention, product, log
    probabilities, against the same steps in 64 bits from the same codes."""
    H, G, hd, P, S, B, V = 4, 2, 32, 150, 40, 7, 500
    dim = H * hd
    rng = np.random.default_rng(12)
    weights = {k: rng.standard_normal(s) / np.sqrt(dim) for k, s in dict(qkv=((H + 2 * G) * hd, dim), o=(dim, dim), head=(V, dim)).items()}
    W = {k: Tensor.from_numpy(ctx, w.astype(f32)).convert(TILES) for k, w in weights.items()}
    wide = {k: stands_for(*parts(t), True) for k, t in W.items()}
    planes = lambda rows: [Tensor.zeros(ctx, rows, hd, DTYPE[cache]) for _ in range(2)]  # noqa: E731
    pk, pv = planes(G * P)
    ck, cv = planes(B * G * S)
    front = Tensor.zeros(ctx, P, hd, TensorDType.Float32).rope_table()
    behind = Tensor.zeros(ctx, S, hd, TensorDType.Float32).rope_table_from(P)
    prompt = Tensor.from_numpy(ctx, rng.standard_normal((P, dim)).astype(f32)).matrix_mul_f8(W["qkv"])
    prompt.qkv_append(Tensor.zeros(ctx, P, dim, TensorDType.Float32), pk, pv, front, H, G, P, [0])
    starts = [0, 5, 30, 11, -1, 2, 36]
    for b in range(B):  # what the texts hold already
        if starts[b] > 0:
            at = [-starts[b]] * B
            at[b] = 0
            old = Tensor.from_numpy(ctx, rng.standard_normal((B * starts[b], (H + 2 * G) * hd)).astype(f32))
            old.qkv_append(Tensor.zeros(ctx, B * starts[b], dim, TensorDType.Float32), ck, cv, behind, H, G, S, at)
    PK, PV = (values(t).reshape(G, P, hd) for t in (pk, pv))
    for step in range(3):
        at = [s + step if s >= 0 else -1 for s in starts]
        x = rng.standard_normal((B, dim)).astype(f32)
        X = Tensor.from_numpy(ctx, x)
        qkv = X.matrix_mul_f8(W["qkv"])
        assert np.abs(qkv.to_numpy() - stands_for(*encode(x, False), False) @ wide["qkv"].T).max() < 1e-5
        q = Tensor.zeros(ctx, B, dim, TensorDType.Float32)
        qkv.qkv_append(q, ck, cv, behind, H, G, S, at)
        K, V_ = (values(t).reshape(B, G, S, hd) for t in (ck, cv))
        seen = q.attn_shared(pk, pv, P, ck, cv, H, G, S, at)
        want, bound = shared_reference(q.to_numpy().astype(f64).reshape(B, 1, H, hd), PK, PV, K, V_, at)
        assert (np.abs(seen.to_numpy().reshape(want.shape) - want) <= bound + 1e-30).all()
        o = seen.matrix_mul_f8(W["o"])
        logits = o.matrix_mul_f8(W["head"])
        logits_want = stands_for(*encode(o.to_numpy(), False), False) @ wide["head"].T
        assert np.abs(logits.to_numpy() - logits_want).max() < 1e-5
        tokens = np.arange(B, dtype=np.int32)[:, None] * 7
        got = [t.to_numpy() for t in logits.token_logprobs(Tensor.from_numpy(ctx, tokens), 0.7, 4)]
        p, h = logprobs_reference(logits.to_numpy(), 0.7)
        assert np.abs(got[0] - np.take_along_axis(p, tokens, 1)).max() < 1e-5 and np.abs(got[1] - h).max() < 1e-4
        assert np.array_equal(got[2], first_of_the_largest(logits.to_numpy(), 4))
