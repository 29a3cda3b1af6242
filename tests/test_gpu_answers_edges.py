"""The operators for many answers to one prompt where memory and streams are concerned: captured into graphs, on other streams and contexts, two calls at once, offsets past
32 bits, operands that share memory."""
import ctypes
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import rllama_amd
import test_gpu_answers as base
from rllama_amd import Context, Tensor, TensorDType
from test_gpu_answers import F8, TILES, decode, encode, first_of_the_largest, logprobs_reference, shared_reference, stands_for
from test_gpu_longctx import EPS16, EPS32, INVALID, STATE, UNSUPPORTED, f16, f32, f64, refused, upload, values
from test_gpu_longctx_edges import hip_runtime

pytestmark = pytest.mark.gpu


class Step:
    """One step of a batch: product of 8 bits, attention behind the prefix, output head, log probabilities; all results have their memory beforehand."""

    def __init__(self, ctx, seed, B=20, n=1, kind="f16", H=8, G=2, hd=64, P=700, S=90, V=900):
        rng = np.random.default_rng(seed)
        self.ctx, self.rng, self.kind, self.at = ctx, rng, kind, (H, G, S)
        self.P, self.starts, self.rows, self.dim = P, [(7 * b) % (S - n) for b in range(B)], B * n, H * hd
        T = {"f16": TensorDType.Float16, "f32": TensorDType.Float32}[kind]
        put = lambda *s: Tensor.from_numpy(ctx, rng.standard_normal(s).astype({"f16": f16, "f32": f32}[kind]))  # noqa: E731
        self.planes = [put(G * P, hd), put(G * P, hd), put(B * G * S, hd), put(B * G * S, hd)]
        self.weights = [Tensor.from_numpy(ctx, (rng.standard_normal(s) / np.sqrt(self.dim)).astype(f32)).convert(TILES) for s in ((H * hd, self.dim), (V, self.dim))]
        zeros = lambda r, c, t: Tensor.zeros(ctx, r, c, t)  # noqa: E731
        self.x, self.q, self.seen = (zeros(self.rows, self.dim, T) for _ in range(3))
        self.codes = zeros(self.rows, self.dim, F8)
        self.logits = zeros(self.rows, V, TensorDType.Float32)
        self.tokens = Tensor.from_numpy(ctx, rng.integers(0, V, (self.rows, 2)).astype(np.int32))
        self.results = dict(logprobs=zeros(self.rows, 2, TensorDType.Float32), entropy=zeros(self.rows, 1, TensorDType.Float32), top_ids=zeros(self.rows, 5, TensorDType.Int32),
                            top_logprobs=zeros(self.rows, 5, TensorDType.Float32))

    def next_input(self):
        new = Tensor.from_numpy(self.ctx, self.rng.standard_normal((self.rows, self.dim)).astype({"f16": f16, "f32": f32}[self.kind]))
        rllama_amd._lib.check(self.ctx._lib.rlh_copy_inplace(self.x._h, new._h))

    def run(self):
        self.x.matrix_mul_f8(self.weights[0], out=self.q)
        self.q.attn_shared(*self.planes[:2], self.P, *self.planes[2:], *self.at, self.starts, out=self.seen)
        self.seen.convert(out=self.codes)
        self.codes.matrix_mul_f8(self.weights[1], out=self.logits)
        self.logits.token_logprobs(self.tokens, 0.8, **self.results)

    def outputs(self):
        return [t.to_numpy() for t in (self.q, self.seen, self.codes, self.logits, *self.results.values())]


SHAPES = [dict(), dict(B=3, kind="f32"), dict(B=70, P=2000), dict(B=4, n=40), dict(B=1, P=64, S=8)]


@pytest.mark.parametrize("shape", SHAPES)
def test_captured_and_replayed(shape):
    """A step captured into a graph and replayed with other inputs, with eager work of the same and of another size in between, is the eager step."""
    ctx = Context(0)
    hip = hip_runtime()
    step, other = Step(ctx, 1, **shape), Step(ctx, 2, B=9)
    step.next_input()
    step.run()  # (work memory)
    ctx.sync()
    stream, graph, ready = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0  # relaxed
        ctx.wait_stream(stream.value)
        step.run()
        ctx.release_stream(stream.value)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        for turn in range(4):
            step.next_input()
            ctx.sync()
            if turn % 2:
                other.next_input()
                other.run()
            step.run()
            want = step.outputs()
            for t in (step.q, step.seen, step.logits, *step.results.values()):  # nothing is left of the eager step
                zero = Tensor.zeros(ctx, t.rows(), t.cols(), t.dtype())
                rllama_amd._lib.check(ctx._lib.rlh_copy_inplace(t._h, zero._h))
            ctx.sync()
            for _ in range(1 + turn):
                assert hip.hipGraphLaunch(ready, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            for got, w in zip(step.outputs(), want):
                assert np.array_equal(got, w)
    finally:
        if ready.value:
            hip.hipGraphExecDestroy(ready)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(stream)
        ctx.close()


def test_work_memory_is_not_allocated_while_captured():
    """Calls that need work memory are refused while the stream is captured, nothing is recorded of them, and they run afterwards."""
    ctx = Context(0)
    hip = hip_runtime()
    ctx.set_option("ATTN_SHARED_FORM", "2")  # (with partial results)
    step = Step(ctx, 3, B=70)
    step.next_input()
    ctx.sync()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        ctx.wait_stream(stream.value)
        refused(STATE, step.x.matrix_mul_f8, step.weights[0], out=step.q)
        refused(STATE, step.q.attn_shared, *step.planes[:2], step.P, *step.planes[2:], *step.at, step.starts, out=step.seen)
        ctx.release_stream(stream.value)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        step.run()
        first = step.outputs()
        step.run()
        assert all(np.array_equal(a, b) for a, b in zip(first, step.outputs()))
    finally:
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(stream)
        ctx.close()


def test_two_contexts_and_two_threads(ctx):
    """Steps of two contexts at once, and of two threads that share one, are what each gives alone."""
    other = Context(0)
    steps = [Step(ctx, 5), Step(ctx, 6, B=40, kind="f32"), Step(other, 7, B=3, n=30), Step(other, 8, B=33)]
    wants = []
    for s in steps:
        s.next_input()
        s.run()
        wants.append(s.outputs())
    errors = []

    def work(s):
        try:
            for _ in range(20):
                s.run()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, want in zip(steps, wants):
        assert all(np.array_equal(a, b) for a, b in zip(s.outputs(), want))
    del steps, s
    other.close()


OTHER_OWNER = """
import numpy as np, torch
torch.cuda.init()  # this process uses the HIP runtime that torch brings
from rllama_amd import Context, Tensor, TensorDType
from test_gpu_answers import decode, encode, logprobs_reference
ctx = Context(0)
side = torch.cuda.Stream()
m, k, n = 24, 272, 500
W = Tensor.from_numpy(ctx, np.random.default_rng(1).standard_normal((n, k)).astype(np.float32)).convert(TensorDType.Float8Tiles)
ctx.sync()
with torch.cuda.stream(side):
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(8):
        big = big @ big * 0.01  # keeps the stream busy while the calls below are queued
    x = torch.randn(m, k, device="cuda")
    y = torch.full((m, n), float("nan"), device="cuda")
    h = torch.full((m, 1), float("nan"), device="cuda")
X, Y, E = (Tensor.from_device(ctx, t.data_ptr(), *t.shape, TensorDType.Float32) for t in (x, y, h))
ctx.wait_stream(side.cuda_stream)
X.matrix_mul_f8(W, out=Y)
Y.token_logprobs(entropy=E)
ctx.release_stream(side.cuda_stream)
with torch.cuda.stream(side):
    z, twice = y * 2, h * 2
side.synchronize()
W32 = W.convert(TensorDType.Float32).to_numpy().astype(np.float64)
codes, scales = encode(x.cpu().numpy(), False)
want = (decode(codes) * scales.astype(np.float64).repeat(128, 1)[:, :k]) @ W32.T
assert np.abs(z.cpu().numpy() / 2 - want).max() < 1e-4
assert np.abs(twice.cpu().numpy() / 2 - logprobs_reference(y.cpu().numpy(), 1.0)[1]).max() < 1e-4
for t in (X, Y, E):
    t.free()
ctx.close()
print("the same")
"""


def test_tensors_of_another_owner_on_another_stream():
    """In a process of its own: torch loads its own HIP runtime, which has to come before the library's."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    r = subprocess.run([sys.executable, "-c", OTHER_OWNER], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "the same" in r.stdout, r.stdout + r.stderr


# -- offsets past 32 bits -----------------------------------------------------------------------------------------------------------------

class Memory:
    """Device memory, as it comes, and tensors over parts of it."""

    def __init__(self, ctx, size):
        self.ctx, self.hip, self.at = ctx, hip_runtime(), ctypes.c_void_p()
        assert self.hip.hipMalloc(ctypes.byref(self.at), ctypes.c_size_t(size)) == 0

    def tensor(self, rows, cols, dtype, offset=0):
        return Tensor.from_device(self.ctx, self.at.value + offset, rows, cols, dtype)

    def put(self, array, offset):
        a = np.ascontiguousarray(array)
        assert self.hip.hipMemcpy(ctypes.c_void_p(self.at.value + offset), a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1) == 0

    def get(self, shape, dtype, offset):
        self.ctx.sync()
        a = np.empty(shape, dtype)
        assert self.hip.hipMemcpy(a.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(self.at.value + offset), ctypes.c_size_t(a.nbytes), 2) == 0
        return a

    def free(self):
        self.ctx.sync()
        assert self.hip.hipFree(self.at) == 0


@pytest.mark.parametrize("n", [1, 40])
def test_planes_longer_than_32_bits(ctx, n):
    """Planes of 17 million positions per head: the second head's, and the third text's, lie 4 GiB and more behind the first one's."""
    G, H, hd, P, B, long = 2, 4, 128, 300, 3, 17_000_000
    row, S = hd * 2, 9_000_000
    rng = np.random.default_rng(3)
    prefix, own = [Memory(ctx, G * long * row) for _ in range(2)], [Memory(ctx, B * G * S * row) for _ in range(2)]
    try:
        at = [60, 7, 33]
        shared, texts = rng.standard_normal((2, G, P, hd)).astype(f16), rng.standard_normal((2, B, G, 120, hd)).astype(f16)
        for i in range(2):
            for g in range(G):
                prefix[i].put(shared[i, g], g * long * row)
                for b in range(B):
                    own[i].put(texts[i, b, g], (b * G + g) * S * row)
        q = rng.standard_normal((B, n, H, hd)).astype(f16)
        planes = [m.tensor(G * long, hd, TensorDType.Float16) for m in prefix] + [m.tensor(B * G * S, hd, TensorDType.Float16) for m in own]
        got = Tensor.from_numpy(ctx, q.reshape(B * n, -1)).attn_shared(*planes[:2], P, *planes[2:], H, G, S, at).to_numpy().astype(f64)
        want, bound = shared_reference(q.astype(f64), *shared.astype(f64), *texts.astype(f64), at)
        assert (np.abs(got.reshape(want.shape) - want) <= bound + 2 * EPS16 * max(np.abs(shared[1]).max(), np.abs(texts[1]).max())).all()
        for t in planes:
            t.free()
    finally:
        for m in prefix + own:
            m.free()


def test_logits_longer_than_32_bits(ctx):
    rows, vocab, known = 33_000, 131_072, 3
    rng = np.random.default_rng(4)
    m = Memory(ctx, rows * vocab * 2)
    try:
        x = rng.standard_normal((known, vocab)).astype(f16)
        m.put(x, (rows - known) * vocab * 2)
        logits = m.tensor(rows, vocab, TensorDType.Float16)
        got = logits.token_logprobs(Tensor.from_numpy(ctx, np.full((rows, 1), vocab - 1, np.int32)), 1.0, 3)
        want, entropy = logprobs_reference(x, 1.0)
        tol = EPS32 * (8 + 2 * np.sqrt(vocab) + 6 * np.abs(want).max() + 6 * np.log(vocab))
        assert (np.abs(got[0].to_numpy()[-known:, 0] - want[:, -1]) <= tol).all()
        assert (np.abs(got[1].to_numpy()[-known:] - entropy) <= EPS32 * (16 + 2 * np.sqrt(vocab)) * (entropy + 8 * np.log(vocab))).all()
        assert np.array_equal(got[2].to_numpy()[-known:], first_of_the_largest(x, 3))
        logits.free()
    finally:
        m.free()


@pytest.mark.parametrize("m,n,k,result", [(70_000, 65_536, 128, "f16"), (70_000, 100, 65_536, "f32"), (1, 40_000, 110_000, "f32"), (40, 40_000, 110_000, "f16")])
def test_products_longer_than_32_bits(ctx, m, n, k, result):
    """Codes of the rows, of the weights, or results of more than 4 GiB: the last rows times the last weights."""
    rng = np.random.default_rng(m + n)
    across, tiles = -(-k // 128), -(-n // 128)
    tail = min(m, 2)
    X, W, Y = Memory(ctx, m * k + m * across * 4), Memory(ctx, n * k + tiles * across * 4), Memory(ctx, m * n * (2 if result == "f16" else 4))
    try:
        kind = {"f16": TensorDType.Float16, "f32": TensorDType.Float32}[result]
        xc, xs = rng.integers(0, 96, (tail, k), dtype=np.uint8) + (128 * rng.integers(0, 2, (tail, k))).astype(np.uint8), rng.uniform(0.001, 0.01, (tail, across)).astype(f32)
        first = (tiles - 1) * 128  # the columns of the last tile
        wc = rng.integers(0, 96, (n - first, k), dtype=np.uint8) + (128 * rng.integers(0, 2, (n - first, k))).astype(np.uint8)
        ws = rng.uniform(0.001, 0.01, (1, across)).astype(f32)
        X.put(xc, (m - tail) * k)
        X.put(xs, m * k + (m - tail) * across * 4)
        W.put(wc, first * k)
        W.put(ws, n * k + (tiles - 1) * across * 4)
        x, w, y = X.tensor(m, k, F8), W.tensor(n, k, TILES), Y.tensor(m, n, kind)
        x.matrix_mul_f8(w, out=y)
        a, b = decode(xc) * xs.astype(f64).repeat(128, 1)[:, :k], decode(wc) * ws.astype(f64).repeat(128, 1)[:, :k]
        want, size = a @ b.T, np.abs(a) @ np.abs(b).T
        got = Y.get((tail, n), {"f16": f16, "f32": f32}[result], (m - tail) * n * (2 if result == "f16" else 4))[:, first:].astype(f64)
        # f32: a rounding per block and per sum of a block; f16 results of many rows: products of a group of eight are cut off 2^-13 below the largest
        tol = size * EPS32 * (across + 140) + (size * 2.0 ** -12 + EPS16 * np.abs(want) if result == "f16" else 0)
        assert (np.abs(got - want) <= tol).all()
        for t in (x, w, y):
            t.free()
    finally:
        for memory in (X, W, Y):
            memory.free()


# -- the form that the estimate does not choose ---------------------------------------------------------------------------------------------

@pytest.fixture(params=["1", "2"])
def form(ctx, request):
    ctx.set_option("ATTN_SHARED_FORM", request.param)
    yield ctx
    ctx.set_option("ATTN_SHARED_FORM", None)


@pytest.mark.parametrize("case", base.SHARED)
@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4")])
def test_both_forms(form, case, kind, cache):
    base.test_attention_behind_a_shared_prefix(form, *case, kind, cache)


@pytest.mark.parametrize("P", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 383, 511, 513, 1025, 3000])
@pytest.mark.parametrize("cache,B", [("f16", 20), ("q4", 20), ("f16", 70)])
def test_both_forms_of_prefixes_of_every_length(form, P, cache, B):
    base.test_prefixes_of_every_length(form, P, "f16", cache, B)


@pytest.mark.parametrize("n,B", [(1, 40), (20, 5), (70, 4)])
def test_both_forms_of_scores_far_apart(form, n, B):
    base.test_scores_far_apart(form, "f16", n, B)


@pytest.mark.parametrize("cache", ["f16", "q4"])
@pytest.mark.parametrize("B,n,group", [(30, 1, 4), (4, 20, 1), (12, 7, 3), (5, 20, 2), (3, 34, 4)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_both_forms_of_values_that_are_not_finite(form, cache, B, n, group, value):
    base.test_values_that_are_not_finite_reach_the_rows_that_see_them(form, "f16", cache, B, n, group, value)


@pytest.mark.parametrize("cache", ["f16", "q4"])
@pytest.mark.parametrize("hd,n,P,starts", [(32, 40, 256, [-40, -40, -99]), (64, 1, 0, [-2] * 40), (128, 50, 0, [-50]), (128, 1, 500, [-1] * 40)])
def test_both_forms_of_nothing_but_padding(form, cache, hd, n, P, starts):
    base.test_nothing_but_padding(form, "f16", cache, hd, n, P, starts)


def test_more_rows_than_a_launch_takes(ctx):
    """Log probabilities of 17 million short rows; attention of more rows than one launch's workgroups have is refused, as are planes whose positions come near 32 bits."""
    rows, vocab = 17_000_000, 16
    rng = np.random.default_rng(9)
    m = Memory(ctx, rows * vocab * 2)
    try:
        known = [0, 2 ** 21 - 1, 2 ** 21, 2 ** 24, rows - 1]
        x = rng.standard_normal((len(known), vocab)).astype(f16)
        for r, at in enumerate(known):
            m.put(x[r], at * vocab * 2)
        logits = m.tensor(rows, vocab, TensorDType.Float16)
        got = logits.token_logprobs(Tensor.from_numpy(ctx, np.full((rows, 1), 3, np.int32)), 1.0, 2)
        want, entropy = logprobs_reference(x, 1.0)
        assert np.abs(got[0].to_numpy()[known, 0] - want[:, 3]).max() < 1e-5 and np.abs(got[1].to_numpy()[known] - entropy).max() < 1e-4
        assert np.array_equal(got[2].to_numpy()[known], first_of_the_largest(x, 2))
        logits.free()
    finally:
        m.free()
    n = 2 ** 27 + 16
    q, out, plane = Memory(ctx, n * 128), Memory(ctx, n * 128), Tensor.zeros(ctx, 64, 32, TensorDType.Float32)
    try:
        Q, Out = q.tensor(n, 32, TensorDType.Float32), out.tensor(n, 32, TensorDType.Float32)
        refused(UNSUPPORTED, Q.attn_shared, None, None, 0, plane, plane, 1, 1, 64, [64 - n], out=Out)
        Q.free(), Out.free()
    finally:
        q.free()
        out.free()
    small = Tensor.zeros(ctx, 1, 32, TensorDType.Float32)
    refused(UNSUPPORTED, small.attn_shared, None, None, 0, plane, plane, 1, 1, 2 ** 31 - 256, [0])
    refused(UNSUPPORTED, small.attn_shared, plane, plane, 2 ** 31 - 256, plane, plane, 1, 1, 64, [0])


# -- nothing rounded but the result ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", ["f16", "q4"])
@pytest.mark.parametrize("H,G,n,B,P", [(8, 2, 1, 4, 300), (8, 2, 1, 40, 900), (4, 2, 50, 3, 700)])
def test_only_the_result_is_rounded_on_request(ctx, cache, H, G, n, B, P):
    """Values around zero, so that the result's own rounding hides nothing, in the forms for few rows, for a batch of single rows and for many rows of each text."""
    hd, S = 64, 80
    rng = np.random.default_rng(P)
    q = rng.standard_normal((B, n, H, hd)).astype(f16)
    planes = [upload(ctx, rng.standard_normal((rows, hd)), cache) for rows in (G * P, G * P, B * G * S, B * G * S)]
    starts = [(5 * b) % (S - n) for b in range(B)]
    wide = [values(t).reshape(-1, P, hd) if i < 2 else values(t).reshape(B, G, S, hd) for i, t in enumerate(planes)]
    want, bound = shared_reference(q.astype(f64), *wide, starts)
    ctx.set_option("ATTN_EXACT", "1")
    try:
        got = Tensor.from_numpy(ctx, q.reshape(B * n, -1)).attn_shared(*planes[:2], P, *planes[2:], H, G, S, starts).to_numpy().astype(f64).reshape(want.shape)
    finally:
        ctx.set_option("ATTN_EXACT", None)
    assert (np.abs(got - want) <= bound + EPS16 * np.abs(want) + 2.0 ** -24).all()


# -- operands that share memory -----------------------------------------------------------------------------------------------------------

def test_results_that_share_memory_are_refused(ctx):
    z = lambda r, c, k=TensorDType.Float32: Tensor.zeros(ctx, r, c, k)  # noqa: E731
    logits, one, ids = z(4, 50), z(4, 1), z(4, 1, TensorDType.Int32)
    refused(INVALID, logits.token_logprobs, ids, 1.0, logprobs=one, entropy=one)
    refused(INVALID, logits.token_logprobs, ids, 1.0, logprobs=one, top_ids=z(4, 1, TensorDType.Int32), top_logprobs=one)
    refused(INVALID, logits.token_logprobs, ids, 1.0, top_ids=ids, top_logprobs=z(4, 1))
    refused(INVALID, one.token_logprobs, entropy=one)
    m = Memory(ctx, 4 * 128 * 8)
    try:
        wide, narrow, tile = m.tensor(4, 128, TensorDType.Float32), m.tensor(4, 128, F8), m.tensor(4, 128, TILES)
        refused(INVALID, wide.convert, out=narrow)
        refused(INVALID, narrow.convert, out=wide)
        refused(INVALID, wide.matrix_mul_f8, Tensor.zeros(ctx, 128, 128, TILES), out=wide)
        refused(INVALID, z(4, 128).matrix_mul_f8, tile, out=m.tensor(4, 4, TensorDType.Float32))
        for t in (wide, narrow, tile):
            t.free()
    finally:
        m.free()
