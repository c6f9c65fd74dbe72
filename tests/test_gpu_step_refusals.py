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


def test_an_append_of_many_sequences():
    """More sequences than one launch carries: a bad one among the last is refused before the first's rows are replaced."""
    from oomllama_b200._lib import OomAttnError
    n = 131
    eng = make_engine(2, 1, [16] * n, kv_dtype="f32")
    k = randn((3, 1, 128), 1).cuda()
    for s in range(n):
        eng.kv_write(0, s, k, -k)
    q, kv = torch.zeros(n, 256, device="cuda"), torch.zeros(n, 128, device="cuda")
    for bad in (4, -1):
        starts = [1] * n
        starts[130] = bad
        with pytest.raises(OomAttnError) as e:
            eng.rope_append(0, list(range(n)), q, kv, kv, starts=starts)
        assert e.value.code == 3
        assert [eng.seq_len(0, s) for s in range(n)] == [3] * n
        assert all(torch.equal(eng.kv_read(0, s)[0][0], k.cpu()[:, 0]) for s in (0, 127, 130))
    eng.rope_append(0, list(range(n)), q, kv, kv, starts=[1] * n)
    assert [eng.seq_len(0, s) for s in range(n)] == [2] * n
    # a sequence of two launches is appended to twice
    eng.rope_append(0, [*range(130), 0], q, kv, kv)
    assert [eng.seq_len(0, s) for s in (0, 1, 129, 130)] == [4, 3, 3, 2]
    eng.sync()
    eng.close()


@pytest.mark.parametrize("step", ["decode", "prefill"])
def test_a_layer_without_room(oracle, step):
    """The second layer's cache is full: the first layer's token is taken back."""
    from oomllama_b200._lib import OomAttnError
    model = _normed_model(oracle, 3)
    eng = make_engine(4, 2, [64, 64], kv_dtype="q4", hidden=512, n_layers=3)
    lens = [[10, 20], [10, 64], [10, 20]]
    for l in range(3):
        for s in range(2):
            eng.set_seq_len(l, s, lens[l][s])
    tokens = torch.ones(2, 20, dtype=torch.int32, device="cuda")
    with pytest.raises(OomAttnError) as e:
        if step == "decode":
            eng.decode_step_q8(model, [0, 1], tokens[:, 0].contiguous())
        else:
            eng.prefill_step_q8(model, [0, 1], tokens)
    assert e.value.code == 3
    assert [[eng.seq_len(l, s) for s in (0, 1)] for l in range(3)] == lens
    eng.sync()
    eng.close()


def test_a_layer_step_whose_scratch_cannot_grow():
    """Captured behind a longer context than any before: the prefill inside is refused, and the append with it."""
    from oomllama_b200._lib import OomAttnError
    H, S = 128, 64
    eng = make_engine(4, 2, [4096], kv_dtype="q4", hidden=H)
    w = [0.1 * randn(s, i).cuda() for i, s in enumerate(((512, H), (256, H), (256, H), (H, 512)))]
    x = randn((1, S, H), 9).cuda()
    eng.attention_forward_with_bias(0, x, *w)
    eng.set_seq_len(0, 0, 3000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(OomAttnError) as e:
            eng.attention_forward_with_bias(0, x, *w)
        assert e.value.code == 8
        x.zero_()
    assert eng.seq_len(0, 0) == 3000
    del graph  # never replayed
    out = eng.attention_forward_with_bias(0, x, *w)
    eng.sync()
    assert eng.seq_len(0, 0) == 3000 + S and torch.isfinite(out).all()
    eng.close()
