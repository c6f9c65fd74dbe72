"""Counts, places and sizes of a call's arguments that do not fit one another: refused before anything is read."""
import pytest
import torch

from helpers import make_engine, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16"])
def test_attention(kv_dtype):
    eng = make_engine(8, 2, [40, 40], kv_dtype=kv_dtype)
    k = randn((40, 2, 128), 1).cuda()
    for s in (0, 1):
        eng.kv_write(0, s, k, k)
    q, q16 = randn((2, 8, 128), 2).cuda(), randn((5, 8, 128), 3, torch.bfloat16).cuda()
    small, lse = torch.empty(1, 8, 128, device="cuda"), torch.empty(15, device="cuda")
    for f in (lambda: eng.decode(0, [0, 1], q, lens=[40]), lambda: eng.decode_packed(0, [0, 1], q, lens=[40, 40, 40]),
              lambda: eng.decode(0, [0, 1], q, out=small), lambda: eng.decode(0, [0, 1], q, with_lse=True, lse=lse),
              lambda: eng.decode(0, [0, 1], q, out=torch.empty(2, 128, 8, device="cuda").transpose(1, 2)),
              lambda: eng.prefill(0, 0, q16, out=small), lambda: eng.rope_q([1, 2], q, out=small)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: eng.decode(0, [0, 1], q, out=torch.empty(2, 8, 128)),
              lambda: eng.decode(0, [0, 1], q, out=torch.empty(2, 8, 128, device="cuda", dtype=torch.bfloat16)),
              lambda: eng.prefill(0, 0, q16, out=torch.empty(5, 8, 128)),
              lambda: eng.prefill(0, 0, q16, out=torch.empty(5, 8, 128, device="cuda", dtype=torch.float16))):
        with pytest.raises(TypeError):
            f()
    # a buffer with room to spare is written as far as the rows go
    want, wide = eng.decode(0, [0, 1], q, lens=iter([40, 7])), torch.full((4, 8, 128), 7.0, device="cuda")
    eng.decode(0, (0, 1), q, lens=[40, 7], out=wide)
    eng.sync()
    assert torch.equal(wide[:2], want) and (wide[2:] == 7).all()
    eng.close()


def test_projections():
    H = 256
    eng = make_engine(2, 1, [40, 40], kv_dtype="bf16", hidden=H)
    x, wq, wk = randn((3, H), 1).cuda(), randn((256, H), 2).cuda(), randn((128, H), 3).cuda()
    with pytest.raises(ValueError):
        eng.qkv_rope_append(0, [0, 1], x, wq, wk, wk)  # three tokens of two sequences
    with pytest.raises(ValueError):
        eng.qkv_rope_append(0, [], x, wq, wk, wk)
    with pytest.raises(TypeError):
        eng.qkv_rope_append(0, [0], x, wq, wk, wk, bq=torch.zeros(256))
    assert eng.seq_len(0, 0) == 0
    eng.qkv_rope_append(0, [0], x, wq, wk, wk)
    eng.sync()
    assert eng.seq_len(0, 0) == 3
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "f32"])
def test_a_layer_step_without_a_hidden_size(kv_dtype):
    from oomllama_b200._lib import OomAttnError, check
    eng = make_engine(2, 1, [40], kv_dtype=kv_dtype, hidden=0)
    p = torch.ones(8, device="cuda").data_ptr()  # an empty tensor has no address
    with pytest.raises(OomAttnError) as e:
        check(eng._ctx, eng._L.oomattn_attention_forward_qk_norm(eng._ctx, 0, 1, 2, p, p, p, p, p, 8, None, None, None,
                                                                 None, p))
    assert e.value.code == 2 and eng.seq_len(0, 0) == 0
    eng.close()


def test_steps(oracle):
    from test_gpu_model_q8 import _model
    model, _ = _model(oracle, 1, 4, 2, 512, 320, 5)
    eng = make_engine(4, 2, [40, 40], kv_dtype="bf16", hidden=512)
    tokens = torch.ones(2, 20, dtype=torch.int32, device="cuda")
    x = randn((2, 512), 1).cuda()
    lay = model.layers[0]
    for ids in ([0], [0, 1, 0], []):
        for f in (lambda: eng.prefill_step_q8(model, ids, tokens), lambda: eng.decode_step_q8(model, ids, tokens[:, 0].contiguous()),
                  lambda: eng.decoder_layer_q8(0, ids, x, lay)):
            with pytest.raises(ValueError):
                f()
    with pytest.raises(ValueError):
        eng.q8_mlp(lay.gate, lay.up, lay.down, x, out=torch.empty(1, 512, device="cuda"))
    assert [eng.seq_len(0, s) for s in (0, 1)] == [0, 0]
    eng.prefill_step_q8(model, [0, 1], tokens)
    eng.decoder_layer_q8(0, (1, 0), x, lay)
    eng.sync()
    assert [eng.seq_len(0, s) for s in (0, 1)] == [21, 21]
    eng.close()
