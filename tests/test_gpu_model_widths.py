"""Models whose layers differ in the width of their MLP."""
import numpy as np
import pytest
import torch

from helpers import make_engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("widths", [(256, 1024), (1024, 256)])
@pytest.mark.parametrize("n_new", [5, 100])
def test_prefill_step_of_unlike_layers(oracle, widths, n_new):
    """The prompt in one step and token by token, over the same bf16 cache: they differ by the prefill's bf16 queries
    (2^-9 of a score, scores up to 8: 1.6e-2 of a weight at most) and f16 weights: 2e-2 of the logits' norm."""
    from test_gpu_model_q8 import _model
    model, _ = _model(oracle, 2, 4, 2, widths[0], 320, 5)
    other, _ = _model(oracle, 1, 4, 2, widths[1], 320, 6)
    model.layers[1] = other.layers[0]
    H = model.layers[0].input_norm.numel()
    engines = [make_engine(4, 2, [128, 128], kv_dtype="bf16", hidden=H, n_layers=2) for _ in range(2)]
    tokens = torch.from_numpy(np.random.default_rng(3).integers(0, 320, (2, n_new)).astype(np.int32)).cuda()
    logits, want = (torch.empty(2, 320, device="cuda") for _ in range(2))
    engines[0].prefill_step_q8(model, [0, 1], tokens, logits=logits)
    for t in range(n_new):
        engines[1].decode_step_q8(model, [0, 1], tokens[:, t].contiguous(), logits=want)
    for e in engines:
        e.sync()
    assert (logits - want).norm() <= 2e-2 * want.norm()
    for e in engines:
        e.close()
