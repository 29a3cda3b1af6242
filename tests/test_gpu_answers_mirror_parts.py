"""The C++ mirror's calls for many answers to one prompt with what may be left out, compared with the same calls from Python."""
import subprocess

import numpy as np
import pytest

from rllama_amd import Tensor, TensorDType, build

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.mark.parametrize("B", [2, 21])
def test_calls_with_parts_left_out(ctx, tmp_path, B):
    rng = np.random.default_rng(B)
    H, G, hd, P, S, V, m, top = 4, 2, 64, 33, 30, 200, 3, 4
    dim, wide = H * hd, (H + 2 * G) * hd
    arrays = [rng.standard_normal(s).astype(f32) for s in ((P, wide), (B, dim), (wide, dim), (V, dim))]
    starts, tokens = [(3 * b) % S for b in range(B)], rng.integers(0, V, (B, m)).astype(np.int32)
    source, result, rest = tmp_path / "in", tmp_path / "out", tmp_path / "parts"
    source.write_bytes(b"".join(a.tobytes() for a in (np.array([H, G, hd, B, P, S, V, m, top], np.int32), *arrays, np.array(starts, np.int32), tokens)))
    r = subprocess.run([build.build_host_answers(), str(source), str(result), str(rest)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr

    prompt, x, w_qkv, w_head = (Tensor.from_numpy(ctx, a) for a in arrays)
    w_qkv, w_head = w_qkv.convert(TensorDType.Float8Tiles), w_head.convert(TensorDType.Float8Tiles)
    pk, pv, ck, cv = (Tensor.zeros(ctx, rows, hd, TensorDType.Float16) for rows in (G * P, G * P, B * G * S, B * G * S))
    prompt.qkv_append(Tensor.zeros(ctx, P, dim, TensorDType.Float32), pk, pv, Tensor.zeros(ctx, P, hd, TensorDType.Float32).rope_table(), H, G, P, [0])
    q = Tensor.zeros(ctx, B, dim, TensorDType.Float32)
    x.matrix_mul_f8(w_qkv).qkv_append(q, ck, cv, Tensor.zeros(ctx, S, hd, TensorDType.Float32).rope_table_from(P), H, G, S, starts)
    out = q.attn_shared(pk, pv, P, ck, cv, H, G, S, starts)
    logits = out.convert(TensorDType.Float8).matrix_mul_f8(w_head, TensorDType.Float32)
    given, best = logits.token_logprobs(Tensor.from_numpy(ctx, tokens)), logits.token_logprobs(None, 0.7, top)
    assert given[2] is None and given[3] is None and best[0] is None
    want = [q.attn_shared(None, None, 0, ck, cv, H, G, S, starts), *given[:2], *best[1:], out.matrix_mul_f8(w_head), out.convert(TensorDType.Float8).matrix_mul_f8(w_head)]
    assert rest.read_bytes() == b"".join(t.to_numpy().tobytes() for t in want)
