"""The operators for long contexts and drafted tokens through the C++ mirror, and 4-bit tensors to the host and back."""
import subprocess

import numpy as np
import pytest

from rllama_amd import Tensor, TensorDType, build

pytestmark = pytest.mark.gpu
f16, f32 = np.float16, np.float32


def test_a_saved_4_bit_tensor_comes_back(ctx):
    rng = np.random.default_rng(3)
    t = Tensor.from_numpy(ctx, rng.standard_normal((37, 96)).astype(f32)).convert(TensorDType.K4BitQuantization)
    saved = t.to_numpy()
    again = Tensor.from_q4(ctx, saved, 37, 96)
    assert np.array_equal(again.to_numpy(), saved)
    assert np.array_equal(again.convert(TensorDType.Float32).to_numpy(), t.convert(TensorDType.Float32).to_numpy())
    for buffer, rows, cols in ((saved[:-1], 37, 96), (saved, 36, 96), (saved.view(np.int8), 37, 96)):
        with pytest.raises(ValueError):
            Tensor.from_q4(ctx, buffer, rows, cols)


@pytest.mark.parametrize("n", [9, 60])
def test_the_cpp_mirror_gives_what_python_gives(ctx, tmp_path, n):
    rng = np.random.default_rng(n)
    H, G, hd, S, window, sinks, V, k = 6, 2, 64, 80, 20, 3, 301, 4
    qkv = rng.standard_normal((n, (H + 2 * G) * hd)).astype(f16)
    norms = [rng.uniform(0.5, 1.5, (1, hd)).astype(f32) for _ in range(2)]
    logits = (rng.standard_normal((k + 1, V)) * 3).astype(f32)
    draft = np.exp(logits[:k] + rng.standard_normal((k, V)) * 0.3)
    draft = (draft / draft.sum(-1, keepdims=True)).astype(f32)
    drafted = draft.argmax(-1).astype(np.int32).reshape(1, k)
    uniforms = rng.random((1, k + 1), dtype=f32)
    arrays = [qkv, *norms, logits, draft, drafted, uniforms]
    source, result = tmp_path / "in", tmp_path / "out"
    source.write_bytes(b"".join(a.tobytes() for a in (np.array([H, G, hd, n, S, window, sinks, V, k], np.int32), *arrays)))
    r = subprocess.run([build.build_host_tensors(), str(source), str(result)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr

    qkv, qn, kn, logits, draft, drafted, uniforms = (Tensor.from_numpy(ctx, a) for a in arrays)
    ck, cv = (Tensor.zeros(ctx, G * S, hd, TensorDType.K4BitQuantization) for _ in range(2))
    q = Tensor.zeros(ctx, n, H * hd, TensorDType.Float16)
    qkv.qkv_append(q, ck, cv, Tensor.zeros(ctx, n, hd, TensorDType.Float32).rope_table(), H, G, S, [0], q_norm=qn, k_norm=kn, eps=1e-5, halves=True, sinks=sinks)
    out = q.attn_window(ck, cv, H, G, S, [0], window=window, sinks=sinks)
    probs = logits.softmax_rows(0.8)
    want = [out, ck, ck.convert(TensorDType.Float32), drafted.verify_draft(probs, draft, uniforms), drafted.verify_draft(probs, None, uniforms)]
    assert result.read_bytes() == b"".join(t.to_numpy().tobytes() for t in want)
    assert np.isfinite(out.to_numpy()).all()
