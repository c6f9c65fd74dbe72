"""The 4-bit KV cache: what it holds, the layout that include/oomattn.h gives, decode and prefill over it, and rows
read back (kv_gather, any cache type), against plain restatements in 64 bits."""
import ctypes
import math

import numpy as np
import pytest
import torch

import q4_ref
from helpers import BF16_RTOL, as_f32_np, assert_close, make_engine, randn

pytestmark = pytest.mark.gpu

# Decode: q and p enter as f16 high + low parts (22 bits), products accumulate in f32.  A score is then off by at most
# about (2^-21 + 2^-21) * sum|q_d k_d| / sqrt(128) <= 2^-20 * 15 for unit normals, an output by twice that times
# max|v| <= 5 : 1.4e-4 in the worst case.  The norm-wise error takes the root mean square instead: 2^-20.
ATOL, RTOL = 1.5e-4, 1e-5


def _filled(n_heads, n_kv, lens, seed=0, dtype=torch.bfloat16, garbage=False, kscale=1.0, vscale=1.0, cap=None):
    eng = make_engine(n_heads, n_kv, [max(1, c) for c in (cap or lens)], kv_dtype="q4", shuffle_seed=seed)
    if garbage:  # NaN scales and offsets in every slot that is not written
        for pool in eng.kv_pool():
            pool.fill_(0xFF)
    ks, vs = [], []
    for s, n in enumerate(lens):
        k = kscale * randn((n, n_kv, 128), seed * 1000 + 2 * s)
        v = vscale * randn((n, n_kv, 128), seed * 1000 + 2 * s + 1)
        k, v = k.to(dtype), v.to(dtype)
        if n:
            eng.kv_write(0, s, k.cuda(), v.cuda())
        ks.append(q4_ref.held(k).transpose(0, 1))
        vs.append(q4_ref.held(v).transpose(0, 1))
    return eng, ks, vs


def _check_decode(eng, n_heads, lens, ks, vs, seed, qscale=1.0, atol=ATOL, rtol=RTOL):
    q = qscale * randn((len(lens), n_heads, 128), seed + 77)
    out, lse = eng.decode(0, list(range(len(lens))), q.cuda(), with_lse=True)
    eng.sync()
    ref = [q4_ref.attend(q[s:s + 1], ks[s], vs[s], [lens[s]]) for s in range(len(lens))]
    want, want_lse = np.concatenate([r[0] for r in ref]), np.concatenate([r[1] for r in ref])
    assert_close(out.cpu().numpy(), want, atol, rtol, what=f"q4 decode {lens}")
    got = lse.cpu().numpy()
    empty = np.isneginf(want_lse)
    np.testing.assert_array_equal(np.isneginf(got), empty)
    np.testing.assert_allclose(got[~empty], want_lse[~empty], rtol=2e-6, atol=1e-5 * max(1.0, qscale))
    return out


# ----------------------------------------------------------------------------------------------- what is held
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [[1], [33], [1, 1, 7, 2, 30], [15, 1, 1, 16, 5]])
def test_cache_holds_the_quantised_rows(dtype, steps):
    """Appends of odd lengths leave exactly the defined codes, neighbours in a slot pair included."""
    n_kv, n = 3, sum(steps)
    eng = make_engine(6, n_kv, [n + 20], kv_dtype="q4")
    for pool in eng.kv_pool():
        pool.fill_(0xFF)
    k, v = (3 * randn((n, n_kv, 128), s).to(dtype) for s in (1, 2))
    at = 0
    for m in steps:
        eng.kv_write(0, 0, k[at:at + m].contiguous().cuda(), v[at:at + m].contiguous().cuda())
        at += m
    eng.sync()
    kc, vc = eng.kv_read(0, 0)
    np.testing.assert_array_equal(kc.numpy(), q4_ref.held(k).transpose(0, 1).numpy())
    np.testing.assert_array_equal(vc.numpy(), q4_ref.held(v).transpose(0, 1).numpy())
    kg, vg = eng.kv_gather(0, [0])
    np.testing.assert_array_equal(kg.cpu().numpy(), q4_ref.held(k).numpy())
    np.testing.assert_array_equal(vg.cpu().numpy(), q4_ref.held(v).numpy())
    eng.close()


def test_special_groups():
    """Constant, zero, tiny, huge, infinite and NaN groups."""
    x = randn((12, 1, 128), 5)
    x[0] = 0.0
    x[1] = -3.3
    x[2] *= 1e-7
    x[3] *= 2e4
    x[4, 0, 5], x[4, 0, 70] = math.inf, -math.inf
    x[5, 0, 40] = math.nan
    x[6, 0, :32] = 1000.0 + 0.01 * x[6, 0, :32]
    x[7] = 3e38 * torch.sign(x[7])
    x[8, 0, 0] = 1e30
    x[9] = -0.0
    x[10] = x[10].half().float() * 2.0 ** -20
    eng = make_engine(2, 1, [12], kv_dtype="q4")
    eng.kv_write(0, 0, x.cuda(), x.flip(0).contiguous().cuda())
    kc, vc = eng.kv_read(0, 0)
    kg, vg = eng.kv_gather(0, [0])
    want, want_v = q4_ref.held(x), q4_ref.held(x.flip(0))
    np.testing.assert_array_equal(kc[0].numpy(), want[:, 0].numpy())
    np.testing.assert_array_equal(vc[0].numpy(), want_v[:, 0].numpy())
    np.testing.assert_array_equal(kg.cpu().numpy(), want.numpy())
    np.testing.assert_array_equal(vg.cpu().numpy(), want_v.numpy())
    assert torch.isnan(kc[0, 5, 32:64]).all() and not torch.isnan(kc[0, 5, :32]).any()
    assert torch.isfinite(kc[0, [3, 4, 7, 8]]).all()
    eng.close()


def test_pool_layout_is_the_documented_one():
    n_kv, n = 2, 37
    eng = make_engine(4, n_kv, [48], kv_dtype="q4", shuffle_seed=3)
    eng.set_block_table(0, [2, 0, 1])
    k, v = randn((n, n_kv, 128), 1), randn((n, n_kv, 128), 2)
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    eng.sync()
    kp, vp = (p.cpu().numpy()[0] for p in eng.kv_pool())
    (kc, ks, ko), (vc, vs, vo) = q4_ref.quantize(k), q4_ref.quantize(v)
    half = lambda chunk, off: float(chunk[off:off + 2].view(np.float16)[0])  # noqa: E731
    for tok in range(n):
        page, r = [2, 0, 1][tok // 16], tok % 16
        for h in range(n_kv):
            kch, vch = kp[page, h], vp[page, h]
            for d in range(0, 128, 3):
                w, t, m = d // 32, d % 32 // 8, d % 8
                word = int(kch[512 * (w // 2) + 32 * r + 8 * t + 4 * (w % 2):][:4].view(np.uint32)[0])
                assert (word >> (4 * m)) & 15 == kc[tok, h, d]
                assert half(kch, 1024 + 16 * r + 2 * w) == ko[tok, h, w]
                assert half(kch, 1024 + 16 * r + 8 + 2 * w) == ks[tok, h, w]
                hh, tt, p, g, m = r // 8, r % 8 // 2, r % 2, d % 32 // 4, d % 4
                piece = int(vch[512 * (w // 2) + 256 * hh + 32 * g + 8 * tt + 4 * (w % 2) + 2 * p:][:2].view(np.uint16)[0])
                assert (piece >> (4 * m)) & 15 == vc[tok, h, d]
                assert half(vch, 1024 + 64 * hh + 16 * tt + 4 * w + 2 * p) == vs[tok, h, w]
                assert half(vch, 1152 + 64 * hh + 16 * tt + 4 * w + 2 * p) == vo[tok, h, w]
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16", "f32"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_gather_ranges(kv_dtype, out_dtype):
    lens = [70, 5, 33]
    eng = make_engine(6, 3, lens, kv_dtype=kv_dtype, shuffle_seed=2)
    kept = []
    for s, n in enumerate(lens):
        k, v = randn((n, 3, 128), 2 * s), randn((n, 3, 128), 2 * s + 1)
        eng.kv_write(0, s, k.cuda(), v.cuda())
        hold = {"q4": q4_ref.held, "bf16": lambda x: x.bfloat16().float(), "f32": lambda x: x}[kv_dtype]
        kept.append((hold(k), hold(v)))
    for ids, starts, n in (([0], [0], 70), ([0, 2, 1], [65, 13, 0], 5), ([1], [4], 1), ([2, 0], [0, 37], 33),
                           ([0, 0], [15, 16], 17), ([0, 1], None, 2), ([0], [70], 0)):
        k, v = eng.kv_gather(0, ids, starts, n, out_dtype=out_dtype)
        at = starts or [0] * len(ids)
        for got, which in ((k, 0), (v, 1)):
            want = torch.cat([kept[s][which][a:a + n] for s, a in zip(ids, at)]).to(out_dtype)
            assert got.dtype == out_dtype
            np.testing.assert_array_equal(as_f32_np(got), want.float().numpy())
    eng.close()


# ----------------------------------------------------------------------------------------------- decode
@pytest.mark.parametrize("heads", [(28, 4), (8, 1), (6, 3), (4, 4), (40, 8), (35, 7)])
@pytest.mark.parametrize("lens", [[1], [2, 15, 16], [17, 31, 32, 33], [0, 63, 64, 65, 0], [513]])
def test_decode_edges(heads, lens):
    eng, ks, vs = _filled(*heads, lens, seed=3, garbage=True)
    _check_decode(eng, heads[0], lens, ks, vs, 3)
    eng.close()


@pytest.mark.parametrize("lens", [[1000, 1, 37, 4097], [20000], [129] * 30 + [2000]])
def test_decode_splits(lens):
    eng, ks, vs = _filled(16, 2, lens, seed=4, dtype=torch.float32, garbage=True)
    _check_decode(eng, 16, lens, ks, vs, 4)
    eng.close()


@pytest.mark.parametrize("qscale,kscale,vscale", [(1e-3, 1.0, 1.0), (0.0, 1.0, 1.0), (30.0, 1.0, 1.0), (1.0, 1e-3, 1.0),
                                                  (1e-4, 1e4, 1.0), (1e4, 1e-4, 1.0), (1.0, 1.0, 1e-3),
                                                  (1.0, 1.0, 1e4), (1e-30, 1.0, 1.0)])
def test_decode_magnitudes(qscale, kscale, vscale):
    """Large and small q, K and V.  Scores that are 30 times larger are off by 30 times as much."""
    lens = [200, 33]
    eng, ks, vs = _filled(8, 2, lens, seed=5, dtype=torch.float32, kscale=kscale, vscale=vscale)
    f = max(1.0, qscale * kscale)
    _check_decode(eng, 8, lens, ks, vs, 5, qscale=qscale, atol=ATOL * f * vscale, rtol=RTOL * f)
    eng.close()


def test_decode_dominant_key_late():
    """A running maximum that jumps in the last tile, and one that never moves again after the first."""
    n = 300
    for at in (0, n - 1):
        k, v = 0.1 * randn((n, 1, 128), 8), randn((n, 1, 128), 9)
        q = randn((1, 4, 128), 10)
        k[at, 0] = 3 * q[0, 1]
        eng = make_engine(4, 1, [n], kv_dtype="q4")
        eng.kv_write(0, 0, k.cuda(), v.cuda())
        out = eng.decode(0, [0], q.cuda())
        eng.sync()
        want, _ = q4_ref.attend(q, q4_ref.held(k).transpose(0, 1), q4_ref.held(v).transpose(0, 1), [n])
        assert_close(out.cpu().numpy(), want, 4 * ATOL, 4 * RTOL, what=f"dominant key {at}")  # scores up to 35
        eng.close()


def test_decode_lens_packed_and_many_rows():
    """Rows of one sequence at lengths of their own, more of them than one launch carries, and the packed form."""
    n, rows = 150, 131
    eng, ks, vs = _filled(4, 2, [n], seed=6)
    q = randn((rows, 4, 128), 61)
    lens = [(7 * i) % (n + 1) for i in range(rows)]
    out = eng.decode(0, [0] * rows, q.cuda(), lens=lens)
    packed = eng.decode_packed(0, [0] * rows, q.cuda(), lens=lens)
    eng.sync()
    want, lse = q4_ref.attend(q, ks[0], vs[0], lens)
    assert_close(out.cpu().numpy(), want, ATOL, RTOL, what="rows at their own lengths")
    np.testing.assert_array_equal(packed[..., :128].cpu().numpy(), out.cpu().numpy())
    got = packed[..., 128].cpu().numpy()
    seen = np.array(lens) > 0
    np.testing.assert_allclose(got[seen], lse[seen], rtol=2e-6, atol=1e-5)
    assert np.isneginf(got[~seen]).all()
    eng.close()


@pytest.mark.parametrize("heads", [(8, 1), (4, 1)])
def test_many_splits_merged_after(heads):
    """One long row of one kv head: more splits than the decode's last CTA joins, f32, packed and bf16 outputs, beside
    a short row, an empty one and one of a single split."""
    lens = [30000, 0, 100, 3001]
    eng, ks, vs = _filled(*heads, lens, seed=15, dtype=torch.float32)
    out = _check_decode(eng, heads[0], lens, ks, vs, 15)
    q = randn((4, heads[0], 128), 15 + 77).cuda()
    packed = eng.decode_packed(0, [0, 1, 2, 3], q)
    np.testing.assert_array_equal(packed[..., :128].cpu().numpy(), out.cpu().numpy())
    for _ in range(3):
        assert torch.equal(eng.decode(0, [0, 1, 2, 3], q), out)
    q16 = randn((2, heads[0], 128), 16, torch.bfloat16)
    want, _ = q4_ref.attend(q16, ks[0], vs[0], [29999, 30000])
    for dt in (torch.float32, torch.bfloat16):
        got = eng.prefill(0, 0, q16.cuda(), out_dtype=dt)
        assert_close(as_f32_np(got), want, ATOL + (2.0 ** -8 if dt == torch.bfloat16 else 0), BF16_RTOL, what="rows")
    eng.close()


def test_nan_reaches_only_rows_that_see_it():
    n = 40
    k, v = randn((n, 2, 128), 1), randn((n, 2, 128), 2)
    v[20, 0, 3] = math.nan   # kv head 0, group 0
    k[39, 1, 100] = math.nan
    eng = make_engine(4, 2, [n], kv_dtype="q4")
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    q = randn((3, 4, 128), 3).cuda()
    out = eng.decode(0, [0, 0, 0], q, lens=[20, 21, 40]).cpu()
    eng.sync()
    assert torch.isfinite(out[0]).all()
    assert torch.isnan(out[1, :2, :32]).all() and torch.isfinite(out[1, :2, 32:]).all() and torch.isfinite(out[1, 2:]).all()
    assert torch.isnan(out[2, 2:]).all()
    eng.close()


def test_decode_static_scratch(lib):
    from oomllama_b200 import _lib
    lens = [1, 530, 0, 4100]
    eng, ks, vs = _filled(28, 4, lens, seed=7)
    q = randn((4, 28, 128), 70).cuda()
    want = eng.decode(0, [0, 1, 2, 3], q)
    eng.sync()
    kp, vp = (p[0] for p in eng.kv_pool())
    # the table again, by the shuffled pages that make_engine dealt out
    pages = [-(-max(1, n) // 16) for n in lens]
    perm = np.random.default_rng(7).permutation(sum(pages))
    bt = torch.full((4, max(pages)), kp.shape[0] - 1, dtype=torch.int32)
    o = 0
    for s, p in enumerate(pages):
        bt[s, :p] = torch.from_numpy(perm[o:o + p].astype(np.int32))
        o += p
    bt, out = bt.cuda(), torch.empty(4, 28, 128, device="cuda")
    err = ctypes.create_string_buffer(256)
    arr = lambda x: (ctypes.c_int32 * len(x))(*x)  # noqa: E731
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731

    def call(k_pool):
        return lib.oomattn_decode_static_scratch(
            0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), _lib.DTYPE_Q4, k_pool, p(vp), kp.shape[0],
            p(bt), bt.shape[1], 28, 4, ctypes.c_float(0.0), 4, arr([0, 1, 2, 3]), arr(lens), p(q), p(out), None, err, 256)

    assert call(ctypes.c_void_p(kp.data_ptr() + 4)) == 1  # a misaligned pool
    assert call(p(kp)) == 0, err.value
    torch.cuda.synchronize()
    assert_close(out.cpu().numpy(), want.cpu().numpy(), 1e-5, 1e-5, what="static scratch")
    eng.close()


# ----------------------------------------------------------------------------------------------- prefill
@pytest.mark.parametrize("heads", [(28, 4), (8, 8), (10, 2), (16, 2), (9, 3), (6, 1), (8, 2)])
@pytest.mark.parametrize("n_new,prefix", [(1, 0), (1, 50), (7, 9), (16, 100), (24, 0), (25, 0), (25, 111), (100, 28), (300, 500),
                                          (24, 3000), (60, 2000)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_prefill(heads, n_new, prefix, out_dtype):
    n = n_new + prefix
    eng, ks, vs = _filled(*heads, [n], seed=8, garbage=True, cap=[n + 100])
    q = randn((n_new, heads[0], 128), 81, torch.bfloat16)
    out, lse = eng.prefill(0, 0, q.cuda(), out_dtype=out_dtype, with_lse=True)
    eng.sync()
    want, want_lse = q4_ref.attend(q, ks[0], vs[0], [prefix + i + 1 for i in range(n_new)])
    # K and V rows rounded to bf16 (2^-8 relative at most, a root mean square of 2^-8 / sqrt(6)) move a score by about
    # 2^-8 / sqrt(6) of its own size and an output by as much again; with few keys nothing averages out: |out| <= 4.5
    # gives 4.5 * (2^-8 (V) + 2^-8 (score) + 2^-8 (bf16 output)) at most
    assert_close(as_f32_np(out), want, 4.5 * 3 * 2.0 ** -8, BF16_RTOL, what=f"prefill {n_new} + {prefix}")
    np.testing.assert_allclose(lse.cpu().numpy(), want_lse, atol=2e-2)
    eng.close()


def test_prefill_grows_and_shrinks():
    """One engine, two sequences of unlike length in turn: what an earlier, longer one left in the scratch stays out."""
    lens = [700, 55, 1500, 49]
    eng, ks, vs = _filled(8, 2, lens, seed=9)
    for s in (0, 1, 2, 3, 1):
        n_new = min(60, lens[s])
        q = randn((n_new, 8, 128), 90 + s, torch.bfloat16)
        out = eng.prefill(0, s, q.cuda())
        eng.sync()
        want, _ = q4_ref.attend(q, ks[s], vs[s], [lens[s] - n_new + i + 1 for i in range(n_new)])
        assert_close(out.cpu().numpy(), want, 4.5 * 2 * 2.0 ** -8, BF16_RTOL, what=f"sequence {s}")
    eng.close()


def test_prefill_blocks():
    n = 600
    eng, ks, vs = _filled(8, 2, [n], seed=10)
    q = randn((n, 8, 128), 100, torch.bfloat16).cuda()
    whole = eng.prefill(0, 0, q)
    part = torch.full_like(whole, 7.0)
    eng.prefill(0, 0, q, out=part, blocks=[(1, 2)])
    eng.sync()
    assert (part[:256] == 7).all() and (part[512:] == 7).all()
    assert_close(part[256:512].cpu().numpy(), whole[256:512].cpu().numpy(), 1e-3, 1e-3, what="block 1")
    eng.close()


# ----------------------------------------------------------------------------------------------- streams, graphs, limits
def test_step_captured_and_replayed():
    """Append and decode of one token in a graph, replayed on other data, beside an eager context."""
    n = 100
    eng, ks, vs = _filled(8, 2, [n], seed=11, cap=[n + 1])
    q, k, v = (torch.zeros(1, h * 128, device="cuda") for h in (8, 2, 2))
    out = torch.empty(1, 8, 128, device="cuda")
    qr = torch.empty(1, 8, 128, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eng.rope_append(0, [0], q, k, v, starts=[n], q_out=qr)  # warm-up
        eng.decode(0, [0], qr, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        eng.rope_append(0, [0], q, k, v, starts=[n], q_out=qr)
        eng.decode(0, [0], qr, out=out)
    for seed in (1, 2, 3):
        new = [randn((1, h * 128), 10 * seed + h) for h in (8, 2, 3)]
        q.copy_(new[0]); k.copy_(new[1]); v.copy_(new[2][:, :256])
        graph.replay()
        torch.cuda.synchronize()
        kr = q4_ref.normed_rope(new[1].view(1, 2, 128), None, None, 0, [n], 1e6, "interleaved")
        kc, vc = eng.kv_read(0, 0)
        assert ((kc[:, n] - kr[0]).abs() <= q4_ref.code_bound(kr[0])).all()
        want, _ = q4_ref.attend(qr.cpu(), kc, vc, [n + 1])
        assert_close(out.cpu().numpy(), want, ATOL, RTOL, what=f"replay {seed}")
    eng.close()


def test_prefill_in_a_capture_needs_its_scratch():
    from oomllama_b200._lib import OomAttnError
    n = 64
    eng, ks, vs = _filled(8, 2, [n], seed=12)
    q = randn((n, 8, 128), 5, torch.bfloat16).cuda()
    out = torch.empty(n, 8, 128, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(OomAttnError) as e:
            eng.prefill(0, 0, q, out=out)
        assert e.value.code == 8
        out.zero_()
    eng.prefill(0, 0, q, out=out)
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.prefill(0, 0, q, out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    np.testing.assert_array_equal(as_f32_np(out), as_f32_np(eager))
    eng.close()


def test_many_splits_captured_and_replayed():
    """A row long enough for the merge by a kernel of its own, behind an append, in a graph: the replays follow the data."""
    n = 9000
    eng, ks, vs = _filled(4, 1, [n], seed=15, cap=[n + 1])
    q, k, v = (randn((1, h * 128), 150 + h).cuda() for h in (4, 1, 2))
    v = v[:, :128].contiguous()
    out, qr = torch.empty(1, 4, 128, device="cuda"), torch.empty(1, 4, 128, device="cuda")

    def step():
        eng.rope_append(0, [0], q, k, v, starts=[n], q_out=qr)
        eng.decode(0, [0], qr, out=out)
        eng.rope_append(0, [0], q, k, v, starts=[n], q_out=qr)  # and again: two merges in a row share the partials
        eng.decode(0, [0], qr, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        q.copy_(randn(q.shape, 160 + seed))
        k.copy_(randn(k.shape, 170 + seed))
        v.copy_(randn(v.shape, 180 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        kc, vc = eng.kv_read(0, 0)
        want, _ = q4_ref.attend(qr.cpu(), kc, vc, [n + 1])
        assert_close(got, want, ATOL, RTOL, what=f"replay {seed}")
    eng.close()


def test_prefill_reports_values_outside_fp16():
    """Many queries: a NaN of V (which a product with a weight of zero would spread) and a q value that fp16 does
    not hold are reported; few queries take both."""
    from oomllama_b200._lib import OomAttnError
    n = 200
    k, v = randn((n, 2, 128), 1), randn((n, 2, 128), 2)
    v[199, 1, 3] = math.nan
    big = torch.ones(100, 4, 128, dtype=torch.bfloat16)
    big[50, 3, 77] = 70000.0
    for vv, q in ((v, big.clamp(-1, 1)), (torch.nan_to_num(v), big)):
        eng = make_engine(4, 2, [n], kv_dtype="q4")
        eng.kv_write(0, 0, k.cuda(), vv.cuda())
        eng.prefill(0, 0, q.cuda())
        with pytest.raises(OomAttnError) as e:
            eng.sync()
        assert e.value.code == 9
        out = eng.prefill(0, 0, q[30:54].cuda())
        eng.sync()
        want, _ = q4_ref.attend(q[30:53], *eng.kv_read(0, 0), [n - 23 + i for i in range(23)])
        assert_close(out[:20].cpu().numpy(), want[:20], ATOL, RTOL, what="rows of neither")
        assert torch.isfinite(out[:23]).all()
        eng.close()


def test_captured_prefill_outlives_larger_ones():
    """Scratch that a larger prefill replaces stays for the graphs that name it: expanded pages and key-split partials."""
    lens = [600, 3000]
    eng, ks, vs = _filled(4, 2, lens, seed=16)
    q = [randn((n, 4, 128), 190 + n, torch.bfloat16).cuda() for n in (60, 400)]
    out = torch.empty(60, 4, 128, device="cuda")
    eng.prefill(0, 0, q[0], out=out)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.prefill(0, 0, q[0], out=out)
    eng.prefill(0, 1, q[1])  # both kinds of scratch grow
    out.zero_()
    graph.replay()
    eng.sync()
    assert torch.equal(out, first)
    want, _ = q4_ref.attend(q[0].cpu(), ks[0], vs[0], [541 + i for i in range(60)])
    assert_close(out.cpu().numpy(), want, 4.5 * 2 * 2.0 ** -8, BF16_RTOL, what="replayed")
    graph = torch.cuda.CUDAGraph()
    from oomllama_b200._lib import OomAttnError
    big = torch.empty(3000, 4, 128, device="cuda", dtype=torch.bfloat16)
    with torch.cuda.graph(graph):
        with pytest.raises(OomAttnError) as e:  # partials of 3000 rows: more than any call so far
            eng.prefill(0, 1, big)
        assert e.value.code == 8
        out.zero_()
    eng.close()


def test_results_repeat_to_the_bit():
    lens = [3000, 17, 900]
    eng, _, _ = _filled(28, 4, lens, seed=13)
    q = randn((3, 28, 128), 131).cuda()
    first = eng.decode(0, [0, 1, 2], q).clone()
    for _ in range(5):
        assert torch.equal(eng.decode(0, [0, 1, 2], q), first)
    eng.close()


def test_bounded_wait():
    """A producer that issues nothing: the waits run out, the status says so, and the context goes on."""
    from oomllama_b200 import _lib
    lens = [100]
    eng, ks, vs = _filled(8, 2, lens, seed=14)
    eng.set_wait_limit(20_000_000)
    eng.set_test_flags(_lib.TEST_DROP_DECODE_COPIES)
    eng.decode(0, [0], randn((1, 8, 128), 1).cuda())
    with pytest.raises(_lib.OomAttnError) as e:
        eng.sync()
    assert e.value.code == 6
    eng.set_test_flags(0)
    _check_decode(eng, 8, lens, ks, vs, 14)
    eng.close()


def test_refusals():
    from oomllama_b200._lib import OomAttnError
    eng = make_engine(4, 2, [40, 40], kv_dtype="q4")
    k = randn((20, 2, 128), 1).cuda()
    eng.kv_write(0, 0, k, k)

    def refused(code, f):
        with pytest.raises(OomAttnError) as e:
            f()
        assert e.value.code == code
        assert eng.seq_len(0, 0) == 20

    q4, kv = torch.zeros(1, 512, device="cuda"), torch.zeros(1, 256, device="cuda")
    refused(3, lambda: eng.kv_gather(0, [0], [10], 11))
    refused(3, lambda: eng.kv_gather(0, [0], [-1], 2))
    refused(3, lambda: eng.kv_gather(0, [5], [0], 1))
    refused(3, lambda: eng.kv_gather(1, [0], [0], 1))
    refused(3, lambda: eng.rope_append(0, [0], q4, kv, kv, starts=[21]))
    refused(3, lambda: eng.rope_append(0, [0], q4, kv, kv, starts=[-1]))
    refused(1, lambda: eng.rope_append(0, [0, 0], q4.repeat(2, 1), kv.repeat(2, 1), kv.repeat(2, 1)))
    refused(3, lambda: eng.kv_write(0, 0, torch.zeros(30, 2, 128, device="cuda"), torch.zeros(30, 2, 128, device="cuda")))
    w = torch.ones(128, device="cuda")
    for eps in (-1.0, math.nan, math.inf):
        refused(1, lambda: eng.rope_append(0, [0], q4, kv, kv, q_norm=w, eps=eps))
    off = torch.ones(132, device="cuda")[1:129]
    refused(1, lambda: eng.rope_append(0, [0], q4, kv, kv, q_norm=off))
    refused(3, lambda: eng.prefill(0, 0, torch.zeros(21, 4, 128, dtype=torch.bfloat16, device="cuda")))
    refused(3, lambda: eng.prefill(0, 1, torch.zeros(3, 4, 128, dtype=torch.bfloat16, device="cuda"),
                                   out_dtype=torch.bfloat16))
    for bad in (torch.ones(127, device="cuda"), torch.ones(128, device="cuda", dtype=torch.bfloat16), torch.ones(128)):
        with pytest.raises((ValueError, TypeError)):
            eng.rope_append(0, [0], q4, kv, kv, k_norm=bad)
    with pytest.raises(ValueError):
        eng.rope_append(0, [0], q4, kv, kv, starts=[1, 2])
    with pytest.raises(ValueError):
        eng.kv_gather(0, [0], [1, 2], 1)
    with pytest.raises(TypeError):
        eng.kv_gather(0, [0], [0], 1, out_dtype=torch.float32, k_out=torch.empty(1, 2, 128, dtype=torch.bfloat16, device="cuda"))
    eng.close()
