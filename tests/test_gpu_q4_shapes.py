"""The 4-bit cache's attention at group sizes and settings beside the usual ones."""
import numpy as np
import pytest
import torch

import q4_ref
from helpers import as_f32_np, assert_close, randn

pytestmark = pytest.mark.gpu

ATOL, RTOL = 1.5e-4, 1e-5  # of the decode: q and weights in 22 bits (tests/test_gpu_q4.py)


@pytest.mark.parametrize("heads", [(3, 1), (9, 3), (12, 2), (2, 2), (64, 8)])
@pytest.mark.parametrize("scale", [None, 0.3, 1e-3])
def test_groups_and_softmax_scales(heads, scale):
    """Decode, packed decode and both forms of the prefill, under a softmax scale of the configuration's."""
    from oomllama_b200 import TurboConfig, TurboEngine
    n_heads, n_kv = heads
    lens = [0, 1, 47, 700]
    eng = TurboEngine(TurboConfig(n_layers=2, hidden_size=0, n_heads=n_heads, n_kv_heads=n_kv, max_seq_len=704, max_seqs=4,
                                  kv_dtype="q4", softmax_scale=scale))
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (randn((n, n_kv, 128), 10 * s + i, torch.bfloat16) for i in (1, 2))
        if n:
            eng.kv_write(1, s, k.cuda(), v.cuda())
        ks.append(q4_ref.held(k).transpose(0, 1))
        vs.append(q4_ref.held(v).transpose(0, 1))
    q = randn((4, n_heads, 128), 5)
    ids = [3, 0, 2, 1]
    out, lse = eng.decode(1, ids, q.cuda(), with_lse=True)
    packed = eng.decode_packed(1, ids, q.cuda())
    want, want_lse = (np.concatenate(x) for x in zip(*(q4_ref.attend(q[i:i + 1], ks[s], vs[s], [lens[s]], scale) for i, s in enumerate(ids))))
    f = max(1.0, (scale or 0) * 128 ** 0.5)  # scores that much larger are off by as much more
    assert_close(out.cpu().numpy(), want, ATOL * f, RTOL * f, what="decode")
    assert torch.equal(packed[..., :128], out) and torch.equal(packed[..., 128], lse)
    empty = np.isneginf(want_lse)
    np.testing.assert_array_equal(np.isneginf(lse.cpu().numpy()), empty)
    np.testing.assert_allclose(lse.cpu().numpy()[~empty], want_lse[~empty], rtol=2e-6, atol=1e-5 * f)
    for n_new in (5, 60):
        q16 = randn((n_new, n_heads, 128), 6, torch.bfloat16)
        want, _ = q4_ref.attend(q16, ks[3], vs[3], [700 - n_new + i + 1 for i in range(n_new)], scale)
        got = as_f32_np(eng.prefill(1, 3, q16.cuda()))
        # 60: K, V and weights in 11 bits, as many roundings as keys weigh in (7 sqrt(3) 2^-11 of a value at most)
        rel = RTOL * f if n_new == 5 else 6e-3 * f
        assert np.linalg.norm(got - want) <= rel * np.linalg.norm(want), n_new
    eng.sync()
    eng.close()


def test_two_contexts_on_two_streams():
    """Steps of two contexts at once, each on a stream of its own: nothing is shared but the caches' own memory."""
    from helpers import make_engine
    lens, engines, streams, wants, outs = [3000, 70], [], [], [], []
    for i in range(2):
        eng = make_engine(8, 2, lens, kv_dtype="q4", shuffle_seed=i)
        ref = []
        for s, n in enumerate(lens):
            k, v = (randn((n, 2, 128), 100 * i + 10 * s + j, torch.bfloat16) for j in (1, 2))
            eng.kv_write(0, s, k.cuda(), v.cuda())
            ref.append((q4_ref.held(k).transpose(0, 1), q4_ref.held(v).transpose(0, 1)))
        eng.sync()
        engines.append(eng)
        streams.append(torch.cuda.Stream())
        q = randn((2, 8, 128), 7 + i)
        q16 = randn((60, 8, 128), 17 + i, torch.bfloat16)
        wants.append((np.concatenate([q4_ref.attend(q[s:s + 1], *ref[s], [lens[s]])[0] for s in (0, 1)]),
                      q4_ref.attend(q16, *ref[0], [2941 + t for t in range(60)])[0]))
        outs.append((q.cuda(), q16.cuda()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append((engines[i].decode(0, [0, 1], outs[i][0]), engines[i].prefill(0, 0, outs[i][1])))
    torch.cuda.synchronize()
    for i in range(2):
        for d, p in got[i]:
            assert torch.equal(d, got[i][0][0]) and torch.equal(p, got[i][0][1])
        assert_close(got[i][0][0].cpu().numpy(), wants[i][0], ATOL, RTOL, what="decode")
        assert_close(got[i][0][1].cpu().numpy(), wants[i][1], 7 * 3 ** 0.5 * 2.0 ** -11, 6e-3, what="prefill")
        engines[i].close()


def test_pages_behind_four_gigabytes():
    """The same rows in a small pool and in the last pages of one whose byte offsets pass 32 bits: equal to the bit."""
    from oomllama_b200 import TurboConfig, TurboEngine
    n, n_kv, n_heads = 700, 8, 32
    cfg = dict(n_layers=1, hidden_size=0, n_heads=n_heads, n_kv_heads=n_kv, max_seq_len=704, max_seqs=1, kv_dtype="q4")
    big_pages = 230_000  # 230000 * 8 * 2560 bytes = 4.7e9
    engines = [TurboEngine(TurboConfig(**cfg, n_pages=p), assign_pages=False) for p in (44, big_pages)]
    order = np.random.default_rng(1).permutation(44)
    for eng, first in zip(engines, (0, big_pages - 44)):
        eng.set_block_table(0, (first + order).tolist())
    q, k, v = (randn((n, h * 128), 1 + h).cuda() for h in (n_heads, n_kv, n_kv))
    w = 1 + 0.1 * randn((128,), 3)
    got = []
    for eng in engines:
        eng.rope_append(0, [0], q, k, v, q_norm=w.cuda(), k_norm=w.cuda(), q_out_dtype=torch.bfloat16)
        eng.rope_append(0, [0], q[:3].contiguous(), k[:3].contiguous(), v[:3].contiguous(), starts=[650])
        qd, qp = randn((1, n_heads, 128), 5).cuda(), randn((70, n_heads, 128), 6, torch.bfloat16).cuda()
        got.append([*eng.kv_gather(0, [0]), *eng.kv_read(0, 0), *eng.decode(0, [0], qd, with_lse=True),
                    *eng.prefill(0, 0, qp, with_lse=True), eng.prefill(0, 0, qp[:5].contiguous())])
        eng.sync()
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert got[0][0].abs().max() > 1
    for eng in engines:
        eng.close()


def test_a_million_tokens():
    """One sequence of 2^20 tokens, zeros but for its last 20 rows: the lse counts the tokens, the values are the last rows'."""
    from oomllama_b200 import TurboConfig, TurboEngine
    n = 1 << 20
    eng = TurboEngine(TurboConfig(n_layers=1, hidden_size=0, n_heads=8, n_kv_heads=1, max_seq_len=n, max_seqs=1, kv_dtype="q4"))
    eng.set_seq_len(0, 0, n - 20)
    k = torch.zeros(20, 1, 128)
    v = randn((20, 1, 128), 1, torch.bfloat16).float()
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    vh = q4_ref.held(v)[:, 0].double()
    q = randn((4, 8, 128), 2, torch.bfloat16)
    out, lse = eng.decode(0, [0] * 4, q.float().cuda(), lens=[n, n - 19, n - 20, 1], with_lse=True)
    want = torch.stack([vh.sum(0) / n, vh[0] / (n - 19), vh[0] * 0, vh[0] * 0])[:, None].expand(-1, 8, -1)
    # all weights are equal: 22 bits each, summed in f32
    assert ((out.cpu().double() - want).abs() <= 1e-5 * want.abs() + 1e-12).all()
    want_lse = torch.tensor([n, n - 19, n - 20, 1]).double().log()[:, None].expand(-1, 8)
    assert ((lse.cpu().double() - want_lse).abs() <= 1e-5).all()
    for n_new in (4, 64):  # by rows, expanded
        qp = randn((n_new, 8, 128), 3, torch.bfloat16)
        out, lse = eng.prefill(0, 0, qp.cuda(), with_lse=True)
        for i in (0, n_new - 1):
            seen = n - n_new + i + 1
            want = vh[:max(0, 20 - (n - seen))].sum(0) / seen
            # expanded: V in 11 bits, the equal weights exact; the tensor core drops 2^-23 of a running sum per 16 keys
            assert ((out[i].cpu().double() - want).abs() <= 1e-3 * want.abs() + 2.0 ** -23 * float(vh.abs().max()) * 20 / n * 64).all()
            assert ((lse[i].cpu().double() - np.log(seen)).abs() <= 2e-5).all()
    eng.sync()
    eng.close()
