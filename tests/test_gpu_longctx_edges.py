"""The long-context operators at the edges of what their numbers and sizes allow, against their definitions in 64 bits."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import rllama_amd
from rllama_amd import Context, Tensor, TensorDType
from test_gpu_longctx import EPS16, INVALID, UNSUPPORTED, attention_reference, f16, f32, f64, refused, test_append as append_test, upload, values

pytestmark = pytest.mark.gpu


def attend(ctx, q, K, V, cache, starts, window=0, sinks=0):
    """q [B, n, H, hd] f16, K and V [B, G, S, hd] -> (what the call gives, the definition's values, the bound of f32 arithmetic, what the planes hold)."""
    B, n, H, hd = q.shape
    G, S = K.shape[1:3]
    ck, cv = upload(ctx, K.reshape(-1, hd), cache), upload(ctx, V.reshape(-1, hd), cache)
    K, V = (values(t).reshape(B, G, S, hd) for t in (ck, cv))
    want, bound, _ = attention_reference(q.astype(f64), K, V, H, G, hd, starts, n, S, window, sinks)
    got = Tensor.from_numpy(ctx, q.reshape(B * n, H * hd)).attn_window(ck, cv, H, G, S, starts, window=window, sinks=sinks)
    return got.to_numpy().astype(f64).reshape(want.shape), want, bound, K, V


# -- groups of 4 bits that span more than f16 does -----------------------------------------------------------------------------

FEW = [(128, 4, 2, 1, 300), (64, 16, 1, 1, 90), (32, 6, 6, 3, 40), (128, 4, 1, 4, 2500)]  # hd, heads, kv heads, rows, positions


@pytest.mark.parametrize("hd,H,G,n,S", FEW)
def test_few_rows_over_wide_groups(ctx, hd, H, G, n, S):
    """Groups from -40000 to 40000, seen and not seen: 15 steps of their scale are more than f16 holds, every value is less."""
    rng = np.random.default_rng(hd + n)
    start = S - n - 5
    q = (rng.standard_normal((1, n, H, hd)) * 2e-4).astype(f16)
    K, V = rng.standard_normal((1, G, S, hd)), rng.standard_normal((1, G, S, hd))
    for x, at in ((K, (3, start, S - 1)), (V, (5, start, S - 2))):
        x[0, :, at, :32] = np.linspace(-40000, 40000, 32)
    got, want, bound, K, V = attend(ctx, q, K, V, "q4", [start])
    # the weights' and the result's rounding to f16
    assert (np.abs(got - want) <= bound + 2 * EPS16 * 40000).all()
    # ... and where nobody sees a wide group, of what is seen
    V[..., :] = np.clip(V, -8, 8)
    V[0, :, S - 2, :32] = np.linspace(-40000, 40000, 32)
    got, want, bound, _, V = attend(ctx, q, K, V, "q4", [start])
    assert (np.abs(got - want) <= bound + 2 * EPS16 * np.abs(V[0, :, :start + n]).max()).all()


@pytest.mark.parametrize("hd,H,G,n,S", FEW)
def test_few_rows_of_large_queries_over_4_bits(ctx, hd, H, G, n, S):
    """The sum of a quarter of a query is more than f16 holds."""
    rng = np.random.default_rng(hd + n)
    big = 65504 / (hd // 4) * 2
    q = (rng.uniform(0.8, 1.2, (1, n, H, hd)) * np.where(rng.random((1, n, H, 1)) < 0.7, big, 1.5)).astype(f16)
    K, V = rng.standard_normal((1, G, S, hd)) * 2 / (big * np.sqrt(hd)), rng.standard_normal((1, G, S, hd))
    got, want, bound, _, V = attend(ctx, q, K, V, "q4", [S - n])
    assert (np.abs(got - want) <= bound + 2 * EPS16 * np.abs(V).max()).all()


# -- values of 4 bits that f16 does not hold ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,H,G,n,S,top", [(128, 32, 8, 600, 620, 65504), (64, 4, 1, 200, 9205, 65504), (32, 40, 40, 500, 600, 65504), (128, 2, 2, 150, 300, 65504),
                                            (128, 4, 2, 1, 300, 65504), (64, 36, 12, 600, 700, 3e5), (128, 8, 2, 200, 2000, 3e5), (64, 8, 2, 3, 500, 3e5)])
def test_values_of_4_bits_beyond_f16(ctx, hd, H, G, n, S, top):
    """Groups from -65504 up: the highest value reads as 65536 or more, whose place in f16 is infinity."""
    rng = np.random.default_rng(hd + n)
    start = S - n - 5
    q = (rng.standard_normal((1, n, H, hd)) * 1e-4).astype(f16)
    K, V = rng.standard_normal((1, G, S, hd)), rng.standard_normal((1, G, S, hd))
    for x, at in ((K, (3, start + n // 2, S - 1)), (V, (5, start + n // 3, S - 2))):
        x[0, :, at, :32] = np.linspace(-65504, top, 32)
    got, want, bound, K, V = attend(ctx, q, K, V, "q4", [start])
    assert max(K.max(), V.max()) > 65520
    over = np.abs(want) > 65520  # (results of few positions among values of 300000)
    assert (got[over] == np.copysign(np.inf, want[over])).all() and np.isfinite(got[~over]).all()
    assert (np.abs(got - want) <= bound + 2 * EPS16 * np.abs(V).max())[~over].all()


# -- 4 bits and few rows: nothing but the weights and the result is rounded ----------------------------------------------------------

@pytest.mark.parametrize("hd,H,G,n,S,window,sinks", [(128, 4, 2, 1, 1000, 0, 0), (128, 32, 4, 2, 700, 0, 0), (64, 8, 1, 2, 5000, 0, 0), (32, 3, 3, 16, 333, 0, 0),
                                                     (128, 8, 8, 5, 3000, 300, 4)])
def test_up_to_16_rows_read_4_bits_exactly(ctx, hd, H, G, n, S, window, sinks):
    rng = np.random.default_rng(hd + n)
    q = (rng.standard_normal((1, n, H, hd)) * 1.5).astype(f16)
    # keys far from zero and large queries: rounding a key's values to f16 would move the scores by more than the rest of the call does
    q, K, V = q * f16(4), rng.standard_normal((1, G, S, hd)) + 8.0, rng.standard_normal((1, G, S, hd))
    got, want, bound, _, V = attend(ctx, q, K, V, "q4", [S - n], window, sinks)
    error = np.abs(got - want)
    assert (error <= bound + 2 * EPS16 * np.abs(V).max()).all()
    # on average: the result's rounding, and the weights', which fall on V independently of each other
    assert error.mean() <= EPS16 * (np.abs(want).mean() + np.sqrt((V * V).mean()))


@pytest.mark.parametrize("hd,H,G,n,T,window", [(128, 4, 4, 1, 1000, 0), (64, 2, 2, 1, 300, 0), (32, 8, 8, 1, 5000, 700), (128, 2, 2, 7, 900, 0)])
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_up_to_16_rows_round_only_their_result(ctx, hd, H, G, n, T, window, cache):
    """Values whose weighted mean is next to zero for every row, so that the result's own rounding hides nothing."""
    rng = np.random.default_rng(T + hd)
    q = np.repeat((rng.standard_normal((1, 1, H, hd)) * 1.5).astype(f16), n, 1)
    K, V = rng.standard_normal((1, G, T, hd)), rng.standard_normal((1, G, T, hd))
    K[:, :, T - n + 1:] = K[:, :, T - n:T - n + 1]  # rows that look at nearly the same
    V[:, :, T - n + 1:] = 0
    _, want, _, _, V0 = attend(ctx, q, K, V, cache, [T - n], window)
    got, want, bound, _, V = attend(ctx, q, K, V0 - want[:, 0, :, None], cache, [T - n], window)
    error, size = np.abs(got - want), np.sqrt((V * V).mean())
    assert (error <= bound + EPS16 * np.abs(want) + 2.0 ** -24).all()
    # on average the scores are off by some roundings of f32, which the weights take on independently of each other; weights rounded to
    # f16 would leave some 2^-15 of V
    assert error.mean() <= EPS16 * np.abs(want).mean() + 2.0 ** -20 * size


@pytest.mark.parametrize("hd,H,G,n,T", [(128, 16, 16, 200, 2000), (64, 20, 20, 200, 3000)])
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_many_rows_round_only_their_result_on_request(ctx, hd, H, G, n, T, cache):
    """The same for calls that otherwise go to the form that rounds weights and values of 4 bits."""
    ctx.set_option("ATTN_EXACT", "1")
    try:
        test_up_to_16_rows_round_only_their_result(ctx, hd, H, G, n, T, 0, cache)
    finally:
        ctx.set_option("ATTN_EXACT", None)


# -- a first token that takes most of the weight -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,H,G,n,T", [(128, 4, 2, 1, 20000), (64, 8, 1, 2, 65700), (128, 8, 2, 60, 12000), (64, 4, 1, 200, 9000), (128, 32, 8, 130, 6000)])
@pytest.mark.parametrize("cache", ["f16", "q4"])
@pytest.mark.parametrize("share", [0.1, 0.02, 0.002])
def test_what_a_dominating_first_token_leaves(ctx, hd, H, G, n, T, cache, share):
    """All but `share` of the weight is on position 0, the rest on thousands of others alike."""
    rng = np.random.default_rng(T)
    S = T + n
    K, V = np.zeros((1, G, S, hd)), np.zeros((1, G, S, hd))
    q = np.zeros((1, n, H, hd))
    q[..., 0] = 8.0
    # keys and values that 4 bits and f16 both hold: fifteen steps of a scale of few bits, sixteenths
    K[:, :, 0, 0] = 15 * np.rint(np.log((1 - share) / share * T) * np.sqrt(hd) / 8.0 / 15 * 32) / 32
    steps = rng.integers(0, 16, hd)
    steps[0::32], steps[1::32] = 0, 15
    V[:, :, 1:] = 0.5 + steps / 16
    ck, cv = upload(ctx, K.reshape(-1, hd), cache), upload(ctx, V.reshape(-1, hd), cache)
    K, V = (values(t).reshape(1, G, S, hd) for t in (ck, cv))
    got = Tensor.from_numpy(ctx, q.reshape(n, -1).astype(f16)).attn_window(ck, cv, H, G, S, [T]).to_numpy().astype(f64).reshape(n, H, hd)
    first = np.exp(8.0 * K[0, :, 0, 0] / np.sqrt(hd))  # [G]; the others' weights are 1
    rest = T + np.arange(n)
    want = (rest[:, None] / (first + rest[:, None]))[..., None] * V[0, None, :, 1]
    want = np.repeat(want, H // G, 1)
    # weights and result are rounded to f16, relative to themselves; sums in f32
    assert (np.abs(got / want - 1) <= 2 * EPS16 + (4 * np.sqrt(S) + 200) * 2.0 ** -24).all()


# -- memory of another owner -----------------------------------------------------------------------------------------------------------------

def hip_runtime():
    """The HIP runtime that the library has loaded."""
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))


def test_freeing_a_wrapped_tensor_waits_for_other_contexts(ctx):
    """The owner may use the memory again: what another context had queued on it is done."""
    other, hip = Context(0), hip_runtime()
    x = np.arange(64 * 96, dtype=f32).reshape(64, 96)
    memory = ctypes.c_void_p()
    put = lambda a: hip.hipMemcpy(memory, a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1)  # noqa: E731
    assert hip.hipMalloc(ctypes.byref(memory), ctypes.c_size_t(x.nbytes)) == 0
    try:
        assert put(x) == 0
        wrapped = Tensor.from_device(ctx, memory.value, 64, 96, TensorDType.Float32)
        a, b, c = (Tensor.zeros(other, 8192, 8192, TensorDType.Float16) for _ in range(3))
        got = Tensor.zeros(other, 64, 96, TensorDType.Float32)
        other.sync()
        for _ in range(60):  # keeps the other context's stream busy for some 50 ms
            rllama_amd._lib.check(ctx._lib.rlh_matrix_mul_inplace_transposed(c._h, a._h, b._h))
        rllama_amd._lib.check(ctx._lib.rlh_copy_inplace(got._h, wrapped._h))
        wrapped.free()
        assert put(np.zeros_like(x)) == 0
        assert np.array_equal(got.to_numpy(), x)
        for t in (a, b, c, got):
            t.free()
    finally:
        other.close()
        assert hip.hipFree(memory) == 0


# -- work memory ------------------------------------------------------------------------------------------------------------------

def test_work_memory_does_not_grow_with_the_text(ctx):
    """A text that gets longer is cut into more pieces; memory for all of them is there from the first cut on."""
    hip = hip_runtime()

    def used():
        free, total = ctypes.c_size_t(), ctypes.c_size_t()
        assert hip.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        return total.value - free.value

    c = Context(0)
    try:
        hd, H, G, n, S = 128, 32, 8, 32, 40000
        ck, cv = (Tensor.zeros(c, G * S, hd, TensorDType.Float16) for _ in range(2))
        q, out = (Tensor.zeros(c, n, H * hd, TensorDType.Float16) for _ in range(2))
        held = []
        for start in (4000, 8000, 16000, 24000, 39000):
            q.attn_window(ck, cv, H, G, S, [start], out=out)
            c.sync()
            held.append(used())
        assert len(set(held)) == 1, held
    finally:
        c.close()


# -- rows of nearly 2^31 entries --------------------------------------------------------------------------------------------------------------

def test_the_longest_rows(ctx):
    """2^31 - 1 entries: the places of the last ones plus four are more than 32 bits hold.  What lies behind a row must not count."""
    hip, V = hip_runtime(), 2 ** 31 - 1
    memory = [ctypes.c_void_p() for _ in range(2)]

    def fill(m, value, count):
        bits = int(np.array(value, f32).view(np.int32))
        assert hip.hipMemsetD32(m, ctypes.c_int(bits), ctypes.c_size_t(count)) == 0 and hip.hipDeviceSynchronize() == 0

    def put(m, at, a):
        a = np.array(a, f32)
        assert hip.hipMemcpy(ctypes.c_void_p(m.value + 4 * at), a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1) == 0

    def get(m, at, count):
        a = np.empty(count, f32)
        assert hip.hipMemcpy(a.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(m.value + 4 * at), ctypes.c_size_t(a.nbytes), 2) == 0
        return a

    try:
        for m, count in zip(memory, (2 * V + 2, V + 1)):
            assert hip.hipMalloc(ctypes.byref(m), ctypes.c_size_t(4 * count)) == 0
        x, p = (Tensor.from_device(ctx, m.value, 1, V, TensorDType.Float32) for m in memory)
        fill(memory[0], -np.inf, V)
        put(memory[0], V - 3, [0.0, 0.0, np.log(2.0), np.nan])  # the last three, and one behind them
        put(memory[1], V - 4, [9.0] * 5)
        for temperature, want in ((1.0, [0, 0.25, 0.25, 0.5, 9]), (0.0, [0, 0, 0, 1, 9])):
            x.softmax_rows(temperature, out=p)
            ctx.sync()
            assert np.allclose(get(memory[1], V - 4, 5), want, rtol=1e-5)
        x.free()
        # a drafted last token that is accepted, and a second row of which only the last entry is possible
        fill(memory[0], 0.0, 2 * V)
        put(memory[0], V - 1, [1.0])
        put(memory[0], 2 * V - 1, [0.5, 1.0])
        target = Tensor.from_device(ctx, memory[0].value, 2, V, TensorDType.Float32)
        drafted = Tensor.from_numpy(ctx, np.array([[V - 1]], np.int32))
        for u in (0.0, 0.9):
            out = drafted.verify_draft(target, None, Tensor.from_numpy(ctx, np.array([[0.5, u]], f32)))
            assert out.to_numpy().tolist() == [[1, V - 1, V - 1]]
    finally:
        ctx.sync()
        for m in memory:
            hip.hipFree(m)


# -- sizes that are refused ---------------------------------------------------------------------------------------------------------------------

def test_positions_next_to_32_bits_are_refused(ctx):
    z = lambda r, c, k=TensorDType.Float16: Tensor.zeros(ctx, r, c, k)  # noqa: E731
    ck, cv, q, qkv, freqs = z(64, 64), z(64, 64), z(2, 64), z(2, 192), z(64, 64, TensorDType.Float32)
    for at in (2 ** 31 - 257, 2 ** 31 - 200, 2 ** 31 - 2):
        refused(INVALID, q.attn_window, ck, cv, 1, 1, 64, [at], window=16)
        refused(INVALID, qkv.qkv_append, q, ck, cv, freqs, 1, 1, 64, [at])
    q.attn_window(ck, cv, 1, 1, 64, [2 ** 31 - 258], window=16)


def test_more_rows_than_a_launch_takes_are_refused(ctx):
    n, hd = 131070, 32
    ck, cv = (Tensor.zeros(ctx, 64, hd, TensorDType.Float32) for _ in range(2))
    for rows in (n, n + 1):
        q, out = (Tensor.zeros(ctx, rows, 8 * hd, TensorDType.Float32) for _ in range(2))
        if rows == n:
            q.attn_window(ck, cv, 8, 1, 64, [64 - n], out=out)
            assert (out.to_numpy() == 0).all()
        else:
            refused(UNSUPPORTED, q.attn_window, ck, cv, 8, 1, 64, [64 - rows], out=out)
    B, G = 256, 256
    plane = Tensor.zeros(ctx, B * G, hd, TensorDType.Float32)
    q, out = (Tensor.zeros(ctx, B, G * hd, TensorDType.Float32) for _ in range(2))
    refused(UNSUPPORTED, q.attn_window, plane, plane, G, G, 1, [0] * B, out=out)


# -- host memory ---------------------------------------------------------------------------------------------------------------------------------

WIDE_TABLE = """
import resource
import numpy as np
from rllama_amd import Context, Tensor, TensorDType
peak = lambda: resource.getrusage(resource.RUSAGE_SELF).ru_maxrss >> 10
ctx = Context(0)
Tensor.zeros(ctx, 3, 128, TensorDType.Float32).rope_table()
t = Tensor.zeros(ctx, 4096, 16384, TensorDType.Float32)
before = peak()
t.rope_table(500.0)
print("MiB more:", peak() - before)
assert peak() - before < 32
last = t.to_numpy()[-1]
angle = 4095 * 500.0 ** (-np.arange(0, 16384, 2) / 16384)
assert np.abs(last.reshape(-1, 2) - np.stack([np.cos(angle), np.sin(angle)], -1)).max() < 1e-7
print("the same")
"""


def test_a_table_of_angles_takes_little_host_memory(ctx):
    """256 MiB of them: formed and sent piece by piece (in a process of its own, for its peak)."""
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    r = subprocess.run([sys.executable, "-c", WIDE_TABLE], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "the same" in r.stdout, r.stdout + r.stderr


# -- appends of many rows: several heads per thread ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,H,G,n,S,sinks,starts", [
    (128, 34, 2, 400, 500, 0, [7]),              # 38 heads of 16 per workgroup and pass: the last pass is not full
    (64, 16, 16, 180, 220, 0, [0, 11, -30, 40]),
    (32, 40, 20, 300, 320, 4, [900, -5]),        # rings
])
@pytest.mark.parametrize("kind,cache", [("f16", "f16"), ("f16", "q4"), ("f32", "f32")])
@pytest.mark.parametrize("halves,norms", [(False, True), (True, True), (True, False)])
def test_append_of_many_rows(ctx, hd, H, G, n, S, sinks, starts, kind, cache, halves, norms):
    append_test(ctx, hd, H, G, n, S, sinks, starts, kind, cache, halves, norms)
