"""4-bit tensors to the host and back."""
import numpy as np
import pytest

from rllama_amd import Tensor, TensorDType

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
