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
