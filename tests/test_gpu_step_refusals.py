"""A refused step leaves the cache as it was: every layer's lengths, whatever the fault lies in."""
import math

import pytest
import torch

from helpers import make_engine, randn

pytestmark = pytest.mark.gpu


def _normed_model(oracle, n_layers):
    from test_gpu_model_q8 import _model
    model, _ = _model(oracle, n_layers, 4, 2, 512, 320, 5)
    for i, w in enumerate(model.layers):
        w.q_norm, w.k_norm = (1 + 0.1 * randn((128,), 2 * i + j) for j in range(2))
        w.q_norm, w.k_norm = w.q_norm.cuda(), w.k_norm.cuda()
    return model


def _bad_eps(w):
    w.eps = math.nan


def _bad_place(w):
    w.k_norm = torch.ones(132, device="cuda")[1:129]


@pytest.mark.parametrize("spoil", [_bad_eps, _bad_place])
@pytest.mark.parametrize("step", ["decode", "prefill"])
def test_a_bad_norm_in_the_last_layer(oracle, step, spoil):
    """The norms of all layers are looked at before the first of them appends."""
    from oomllama_b200._lib import OomAttnError
    model = _normed_model(oracle, 3)
    eng = make_engine(4, 2, [64, 64], kv_dtype="q4", hidden=512, n_layers=3)
    tokens = torch.randint(0, 320, (2, 24), generator=torch.Generator().manual_seed(1)).int().cuda()
    eng.prefill_step_q8(model, [0, 1], tokens)
    eng.sync()
    spoil(model.layers[2])
    with pytest.raises(OomAttnError) as e:
        if step == "decode":
            eng.decode_step_q8(model, [0, 1], tokens[:, 0].contiguous())
        else:
            eng.prefill_step_q8(model, [0, 1], tokens)
    assert e.value.code == 1
    assert [[eng.seq_len(l, s) for s in (0, 1)] for l in range(3)] == [[24, 24]] * 3
    eng.sync()
    eng.close()
