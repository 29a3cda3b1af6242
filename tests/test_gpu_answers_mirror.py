"""The operators for many answers to one prompt through the C++ mirror."""
import subprocess

import numpy as np
import pytest

from rllama_amd import Tensor, TensorDType, build

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.mark.parametrize("B", [3, 40])
def test_the_cpp_mirror_gives_what_python_gives(ctx, tmp_path, B):
    rng = np.random.default_rng(B)
    H, G, hd, P, S, V, m, top = 6, 2, 32, 150, 40, 301, 2, 7
    dim, wide = H * hd, (H + 2 * G) * hd
    arrays = [rng.standard_normal(s).astype(f32) for s in ((P, wide), (B, dim), (wide, dim), (V, dim))]
    starts, tokens = [b % S for b in range(B)], rng.integers(0, V, (B, m)).astype(np.int32)
    source, result = tmp_path / "in", tmp_path / "out"
    source.write_bytes(b"".join(a.tobytes() for a in (np.array([H, G, hd, B, P, S, V, m, top], np.int32), *arrays, np.array(starts, np.int32), tokens)))
    r = subprocess.run([build.build_host_answers(), str(source), str(result)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr

    prompt, x, w_qkv, w_head = (Tensor.from_numpy(ctx, a) for a in arrays)
    w_qkv, w_head = w_qkv.convert(TensorDType.Float8Tiles), w_head.convert(TensorDType.Float8Tiles)
    pk, pv, ck, cv = (Tensor.zeros(ctx, rows, hd, TensorDType.Float16) for rows in (G * P, G * P, B * G * S, B * G * S))
    prompt.qkv_append(Tensor.zeros(ctx, P, dim, TensorDType.Float32), pk, pv, Tensor.zeros(ctx, P, hd, TensorDType.Float32).rope_table(), H, G, P, [0])
    q = Tensor.zeros(ctx, B, dim, TensorDType.Float32)
    x.matrix_mul_f8(w_qkv).qkv_append(q, ck, cv, Tensor.zeros(ctx, S, hd, TensorDType.Float32).rope_table_from(P), H, G, S, starts)
    out = q.attn_shared(pk, pv, P, ck, cv, H, G, S, starts)
    logits = out.convert(TensorDType.Float8).matrix_mul_f8(w_head, TensorDType.Float32)
    want = [out, w_head, logits, *logits.token_logprobs(Tensor.from_numpy(ctx, tokens), 0.7, top)]
    assert result.read_bytes() == b"".join(t.to_numpy().tobytes() for t in want)
    assert all(np.isfinite(t.to_numpy()).all() for t in (out, logits))
