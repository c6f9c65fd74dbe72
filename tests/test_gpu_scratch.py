"""The scratch of a context as it grows: how much it holds, and that captured graphs keep theirs."""
import pytest
import torch

from helpers import make_engine, randn

pytestmark = pytest.mark.gpu


def _free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("kv_dtype", ["bf16", "q4"])
def test_growth_without_graphs_holds_one_block(kv_dtype):
    """Prompts of rising length: where nothing was captured, the scratch is what the largest of them needs, not that
    and every smaller one's besides."""
    H, hq, hkv = 128, 28, 4
    sizes = [2048, 4096, 8192]
    eng = make_engine(hq, hkv, [sizes[-1]], kv_dtype=kv_dtype, hidden=H)
    w = [0.1 * randn((h * 128, H), h).cuda() for h in (hq, hkv, hkv)]
    xs = [randn((n, H), n).cuda() for n in sizes]
    q = torch.empty(sizes[-1], hq, 128, device="cuda")
    del q
    torch.cuda.empty_cache()
    before = _free()
    for x in xs:
        eng.reset()
        eng.qkv_rope_append(0, [0], x, *w)
        eng.sync()
        torch.cuda.empty_cache()
    # the largest call's projections, and its operands' bf16 planes (x and one weight matrix, two of each)
    need = sizes[-1] * (hq + 2 * hkv) * 128 * 4 + 2 * 2 * H * (sizes[-1] + hq * 128)
    assert before - _free() <= need + (16 << 20)
    eng.close()


def test_growth_with_little_memory_left():
    """Scratch that grows step by step asks for half as much again; where only the need itself is left, for that."""
    hq, hkv, n = 8, 8, 65536
    eng = make_engine(hq, hkv, [n], kv_dtype="q4")
    q = randn((60, hq, 128), 1, torch.bfloat16).cuda()
    out = torch.empty(60, hq, 128, device="cuda")
    eng.set_seq_len(0, 0, 4096)
    eng.prefill(0, 0, q, out=out)
    eng.set_seq_len(0, 0, n)
    need = 2 * n * hkv * 128 * 2  # fp16 rows of K and V: 256 MB
    hog = torch.empty(_free() - need - need // 4, dtype=torch.uint8, device="cuda")
    try:
        eng.prefill(0, 0, q, out=out)
        eng.sync()
    finally:
        del hog
        torch.cuda.empty_cache()
    assert (out == 0).all()  # of a cache that holds zeros
    eng.close()


def _captured(f):
    f()  # the scratch of this size
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    return graph


def test_graphs_outlive_larger_calls(oracle):
    """A linear, a Q8 linear, an argmax, an MLP and a decode step in graphs; then each kind of scratch grows; the replays
    give what they gave."""
    from test_gpu_model_q8 import _model
    model, _ = _model(oracle, 2, 4, 2, 512, 320, 5)
    eng = make_engine(4, 2, [64, 400, 400], kv_dtype="bf16", hidden=512, n_layers=2)
    x, w = randn((40, 512), 1).cuda(), randn((256, 512), 2).cuda()
    lay = model.layers[0]
    outs = {"linear": torch.empty(40, 256, device="cuda"), "q8": torch.empty(5, lay.gate.rows, device="cuda"),
            "mlp": torch.empty(3, 512, device="cuda"), "logits": torch.empty(1, 320, device="cuda")}
    tokens = torch.tensor([7], dtype=torch.int32, device="cuda")
    nxt = torch.empty(1, dtype=torch.int32, device="cuda")

    def step():
        for layer in range(2):
            eng.set_seq_len(layer, 0, 20)
        eng.decode_step_q8(model, [0], tokens, next_tokens=nxt, logits=outs["logits"])

    calls = [lambda: eng.linear(x, w, out=outs["linear"]), lambda: eng.q8_linear(lay.gate, x[:5], out=outs["q8"]),
             lambda: eng.q8_mlp(lay.gate, lay.up, lay.down, x[:3], out=outs["mlp"]), step]
    graphs = [_captured(f) for f in calls]
    eng.sync()
    first = {k: t.clone() for k, t in outs.items()}
    # larger ones of every kind
    big = randn((700, 512), 3).cuda()
    eng.linear(big, w)
    eng.q8_linear(lay.gate, big)
    eng.q8_linear(lay.gate, big[:16])
    eng.q8_mlp(lay.gate, lay.up, lay.down, big)
    eng.prefill_step_q8(model, [1, 2], torch.ones(2, 300, dtype=torch.int32, device="cuda"))
    eng.decode_step_q8(model, [1, 2], torch.ones(2, dtype=torch.int32, device="cuda"))
    fill = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")  # what freed blocks would have become
    for t in outs.values():
        t.fill_(-1)
    for g in graphs:
        g.replay()
    eng.sync()
    for k, t in outs.items():
        assert torch.equal(t, first[k]), k
    del fill, graphs
    eng.close()


def test_a_capture_that_would_grow_is_refused(oracle):
    from test_gpu_model_q8 import _model
    from oomllama_b200._lib import OomAttnError
    model, _ = _model(oracle, 1, 4, 2, 512, 320, 5)
    eng = make_engine(4, 2, [64], kv_dtype="bf16", hidden=512)
    lay, x, w = model.layers[0], randn((100, 512), 1).cuda(), randn((64, 512), 2).cuda()
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        for f in (lambda: eng.linear(x, w), lambda: eng.q8_linear(lay.gate, x[:2]),
                  lambda: eng.q8_mlp(lay.gate, lay.up, lay.down, x), lambda: eng.argmax(x)):
            with pytest.raises(OomAttnError) as e:
                f()
            assert e.value.code == 8
        y.add_(1)
    graph.replay()
    eng.q8_linear(lay.gate, x[:2])
    eng.sync()
    assert (y == 1).all()
    eng.close()
