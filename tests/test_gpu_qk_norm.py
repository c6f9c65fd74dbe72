"""Bias, a norm of every q and k head, rotation and the paged append in one pass, into each cache type, alone and in
the layer and model steps that call it, against a restatement in 64 bits."""
import numpy as np
import pytest
import torch

import q4_ref
from helpers import BF16_RTOL, as_f32_np, assert_close, make_engine, randn

pytestmark = pytest.mark.gpu

# f32: the sum of 128 squares, root, division and three products, each within 2^-24, and the rotation's two products
# and sum: under 12 roundings of 2^-24 relative to the head's largest value (|y| <= 1.5 sqrt(128)).
F32 = 12 * 2.0 ** -24 * 17


def _inputs(T, n_heads, n_kv, dtype, seed, bias):
    q, k, v = (1.7 * randn((T, h * 128), seed + i, dtype) for i, h in enumerate((n_heads, n_kv, n_kv)))
    q, k, v = (x.to(dtype) for x in (q, k, v))
    b = [0.3 * randn((h * 128,), seed + 5 + i) if bias else None for i, h in enumerate((n_heads, n_kv, n_kv))]
    w = [1 + 0.2 * randn((128,), seed + 9 + i) for i in range(2)]
    return q, k, v, b, w


def _cu(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16", "f32"])
@pytest.mark.parametrize("variant,theta", [("interleaved", 1e6), ("split_half", 5e5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("heads", [(28, 4), (6, 3), (5, 1)])
def test_append(kv_dtype, variant, theta, dtype, bias, heads):
    n_heads, n_kv = heads
    prefix, n_new, eps = [0, 33, 2000], 5, 1e-5
    eng = make_engine(n_heads, n_kv, [p + n_new for p in prefix], kv_dtype=kv_dtype, variant=variant, theta=theta)
    for s, p in enumerate(prefix):
        eng.set_seq_len(0, s, p)
    T = len(prefix) * n_new
    q, k, v, b, w = _inputs(T, n_heads, n_kv, dtype, 20, bias)
    pos = np.concatenate([np.arange(p, p + n_new) for p in prefix])
    got = eng.rope_append(0, [0, 1, 2], q.cuda(), k.cuda(), v.cuda(), *map(_cu, b), q_out_dtype=dtype,
                          q_norm=w[0].cuda(), k_norm=w[1].cuda(), eps=eps)
    eng.sync()
    qr = q4_ref.normed_rope(q.view(T, n_heads, 128), b[0], w[0], eps, pos, theta, variant)
    kr = q4_ref.normed_rope(k.view(T, n_kv, 128), b[1], w[1], eps, pos, theta, variant)
    vr = v.view(T, n_kv, 128).double() + (0 if b[2] is None else b[2].double().view(-1, 128))
    half = 2.0 ** -8  # half a step of bf16, relative to the value
    assert got.dtype == dtype
    err = (got.cpu().double() - qr).abs()
    assert (err <= F32 + (half * qr.abs() if dtype == torch.bfloat16 else 0)).all(), err.max()
    ks, vs = eng.kv_gather(0, [0, 1, 2], prefix, n_new)
    ks, vs = ks.cpu().double(), vs.cpu().double()
    if kv_dtype == "q4":
        assert ((ks - kr).abs() <= q4_ref.code_bound(kr)).all()
        vf = v.view(T, n_kv, 128).float() + (0 if b[2] is None else b[2].view(-1, 128))
        np.testing.assert_array_equal(vs.numpy(), q4_ref.held(vf).double().numpy())
        # nearly all codes are the ones of the exact rows (a border may fall to either side)
        same = (ks - q4_ref.held(kr.float()).double()).abs() <= 2e-3
        assert same.double().mean() > 0.999
    else:
        r = half if kv_dtype == "bf16" else 0.0
        assert ((ks - kr).abs() <= F32 + r * kr.abs()).all()
        assert ((vs - vr).abs() <= 2.0 ** -23 * vr.abs() + r * vr.abs()).all()
    assert [eng.seq_len(0, s) for s in range(3)] == [p + n_new for p in prefix]
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16", "f32"])
@pytest.mark.parametrize("n_new", [1, 2, 3, 16, 31])
@pytest.mark.parametrize("norm", [True, False])
def test_starts_give_up_rows(kv_dtype, n_new, norm):
    """Drafts replaced from a slot on: the rows before it stay, those behind it are the new ones, alone and in a batch
    where every sequence starts on its own parity."""
    n, n_kv, starts = 60, 2, [7, 12, 60, 0]
    eng = make_engine(4, n_kv, [n + 40] * 4, kv_dtype=kv_dtype)
    for s in range(4):
        k = randn((n, n_kv, 128), s).cuda()
        eng.kv_write(0, s, k, -k)
    before = [eng.kv_read(0, s) for s in range(4)]
    q, k, v, _, w = _inputs(4 * n_new, 4, n_kv, torch.float32, 40, False)
    eng.rope_append(0, [0, 1, 2, 3], q.cuda(), k.cuda(), v.cuda(), k_norm=w[1].cuda() if norm else None, starts=starts)
    eng.sync()
    for s, at in enumerate(starts):
        assert eng.seq_len(0, s) == at + n_new
        kc, vc = eng.kv_read(0, s)
        np.testing.assert_array_equal(as_f32_np(kc[:, :at]), as_f32_np(before[s][0][:, :at]))
        np.testing.assert_array_equal(as_f32_np(vc[:, :at]), as_f32_np(before[s][1][:, :at]))
        rows = slice(s * n_new, (s + 1) * n_new)
        kr = q4_ref.normed_rope(k[rows].view(n_new, n_kv, 128), None, w[1] if norm else None, 1e-6, np.arange(at, at + n_new), 1e6,
                                "interleaved")
        bound = q4_ref.code_bound(kr) if kv_dtype == "q4" else F32 + (2.0 ** -8 * kr.abs() if kv_dtype == "bf16" else 0)
        assert ((kc[:, at:].double().transpose(0, 1) - kr).abs() <= bound).all()
        hold = {"q4": q4_ref.held, "bf16": lambda x: x.bfloat16().float(), "f32": lambda x: x}[kv_dtype]
        np.testing.assert_array_equal(as_f32_np(vc[:, at:]).transpose(1, 0, 2),
                                      hold(v[rows].view(n_new, n_kv, 128)).numpy())
        # what lay behind is still there for a sequence that is lengthened again
        eng.set_seq_len(0, s, n + n_new)
        kc, _ = eng.kv_read(0, s)
        if at + n_new < n:
            np.testing.assert_array_equal(as_f32_np(kc[:, at + n_new:n]), as_f32_np(before[s][0][:, at + n_new:]))
    eng.close()


def test_one_side_only_and_rope_q():
    n_heads, n_kv = 12, 2
    eng = make_engine(n_heads, n_kv, [16, 16], kv_dtype="f32", variant="split_half", theta=5e5, max_seq_len=5000)
    q, k, v, b, w = _inputs(2, n_heads, n_kv, torch.float32, 60, True)
    norm_q = eng.rope_append(0, [0, 1], q.cuda(), k.cuda(), v.cuda(), *map(_cu, b), q_norm=w[0].cuda())
    kc, _ = eng.kv_gather(0, [0, 1], None, 1)
    kr = q4_ref.normed_rope(k.view(2, n_kv, 128), b[1], None, 0, [0, 0], 5e5, "split_half")
    assert ((kc.cpu().double() - kr).abs() <= F32).all()
    assert torch.equal(norm_q, eng.rope_q([0, 0], q.cuda(), b[0].cuda(), q_norm=w[0].cuda()))
    far = eng.rope_q([4999, 17], q.cuda(), b[0].cuda(), q_norm=w[0].cuda(), eps=0.5)
    want = q4_ref.normed_rope(q.view(2, n_heads, 128), b[0], w[0], 0.5, [4999, 17], 5e5, "split_half")
    assert ((far.cpu().double() - want).abs() <= F32).all()
    eng.close()


def test_zero_rows_and_eps():
    """A head of zeros has no direction: eps keeps it zero; with eps = 0 it is NaN, as 0 / 0."""
    eng = make_engine(4, 4, [16], kv_dtype="f32")
    q = torch.zeros(1, 512, device="cuda")
    q[0, 128:] = randn((384,), 1).cuda()
    w = torch.ones(128, device="cuda")
    a = eng.rope_append(0, [0], q, q, q, q_norm=w, k_norm=w, eps=1e-6)
    assert (a[0, 0] == 0).all() and torch.isfinite(a).all()
    a = eng.rope_append(0, [0], q, q, q, q_norm=w, k_norm=w, eps=0.0)
    assert torch.isnan(a[0, 0]).all() and torch.isfinite(a[0, 1:]).all()
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_layer_step(kv_dtype, norm):
    """attention_forward: a prompt, a second chunk and single tokens of a batch, with the heads' norms.  The reference
    recomputes the whole sequence from the rows that the cache holds."""
    H, n_heads, n_kv, B, eps, theta = 256, 8, 2, 2, 1e-6, 1e6
    if kv_dtype == "bf16" and not norm:
        pytest.skip("covered by the layer tests that were there")
    eng = make_engine(n_heads, n_kv, [64] * B, kv_dtype=kv_dtype, hidden=H)
    wq, wk, wv, wo = (0.08 * randn(s, i) for i, s in enumerate(((n_heads * 128, H), (n_kv * 128, H), (n_kv * 128, H),
                                                                 (H, n_heads * 128))))
    bq, bk, bv = (0.2 * randn((h * 128,), 10 + i) for i, h in enumerate((n_heads, n_kv, n_kv)))
    w = [1 + 0.2 * randn((128,), 20 + i) if norm else None for i in range(2)]
    at = 0
    for S in (20, 18, 1, 3, 1):
        x = randn((B, S, H), 100 + at)
        out = eng.attention_forward_with_bias(0, *(t.cuda() for t in (x, wq, wk, wv, wo, bq, bk, bv)), q_norm=_cu(w[0]),
                                              k_norm=_cu(w[1]), eps=eps).cpu()
        eng.sync()
        for b in range(B):
            pos = np.arange(at, at + S)
            xd = x[b].double()
            q = q4_ref.normed_rope((xd @ wq.double().T).view(S, n_heads, 128), bq, w[0], eps, pos, theta, "interleaved")
            k = q4_ref.normed_rope((xd @ wk.double().T).view(S, n_kv, 128), bk, w[1], eps, pos, theta, "interleaved")
            v = (xd @ wv.double().T + bv.double()).view(S, n_kv, 128)
            kc, vc = eng.kv_read(0, b)
            for got, want in ((kc, k), (vc, v)):
                got = got[:, at:].double().transpose(0, 1)
                bound = q4_ref.code_bound(want) if kv_dtype == "q4" else 2.0 ** -8 * want.abs()
                assert ((got - want).abs() <= bound + 2e-4 * want.abs().max()).all()
            o, _ = q4_ref.attend(q, kc.float(), vc.float(), [at + i + 1 for i in range(S)])
            want = torch.from_numpy(o).reshape(S, -1) @ wo.double().T
            # the attention output is within the bf16 path's relative bound, o_proj adds 1e-4
            assert_close(out[b].numpy(), want.numpy(), 2e-2 * float(want.abs().max()), BF16_RTOL, what=f"rows {at}")
        at += S
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16"])
def test_qkv_rope_append(kv_dtype):
    """The projections in front: GEMV sizes and above, f32 and bf16 weights."""
    H, n_heads, n_kv = 128, 4, 2
    for T, wdt in ((1, torch.float32), (3, torch.float32), (2, torch.bfloat16), (20, torch.float32), (20, torch.bfloat16)):
        eng = make_engine(n_heads, n_kv, [32], kv_dtype=kv_dtype, hidden=H)
        x = randn((T, H), T)
        wq, wk, wv = ((0.1 * randn((h * 128, H), 3 + i)).to(wdt) for i, h in enumerate((n_heads, n_kv, n_kv)))
        nw = [1 + 0.2 * randn((128,), 30 + i) for i in range(2)]
        got = eng.qkv_rope_append(0, [0], x.cuda(), wq.cuda(), wk.cuda(), wv.cuda(), q_norm=nw[0].cuda(),
                                  k_norm=nw[1].cuda())
        eng.sync()
        q = q4_ref.normed_rope((x.double() @ wq.double().T).view(T, n_heads, 128), None, nw[0], 1e-6, np.arange(T), 1e6,
                               "interleaved")
        k = q4_ref.normed_rope((x.double() @ wk.double().T).view(T, n_kv, 128), None, nw[1], 1e-6, np.arange(T), 1e6,
                               "interleaved")
        # the linear is within 1e-4 of the product at unit scale, here normed to unit scale
        assert_close(got.cpu().numpy(), q.numpy(), 5e-4, 1e-4, what=f"q of {T} tokens")
        kc, _ = eng.kv_gather(0, [0])
        bound = q4_ref.code_bound(k) if kv_dtype == "q4" else 2.0 ** -8 * k.abs()
        assert ((kc.cpu().double() - k).abs() <= bound + 5e-4).all()
        eng.close()


def _composed(eng, model, ids, tokens, n_new):
    """A model pass by the engine's single operations: logits [B, vocab] of every sequence's last token."""
    B, H = len(ids), eng.config.hidden_size
    x = eng.embed_q8(model.embed, tokens.reshape(-1))
    for i, w in enumerate(model.layers):
        h = eng.rmsnorm(x, w.input_norm, w.eps)
        q, k, v = (eng.q8_linear(m, h, b) for m, b in ((w.q, w.bq), (w.k, w.bk), (w.v, w.bv)))
        qr = eng.rope_append(i, ids, q, k, v, q_norm=w.q_norm, k_norm=w.k_norm, eps=w.eps,
                             q_out_dtype=torch.float32 if n_new == 1 else torch.bfloat16)
        if n_new == 1:
            att = eng.decode(i, ids, qr)
        else:
            att = torch.cat([eng.prefill(i, s, qr[b * n_new:(b + 1) * n_new].contiguous()) for b, s in enumerate(ids)])
        x = x + eng.q8_linear(w.o, att.view(-1, w.o.cols))
        x = eng.q8_mlp(w.gate, w.up, w.down, eng.rmsnorm(x, w.post_norm, w.eps), residual=x)
    last = x.view(B, n_new, H)[:, -1].contiguous()
    return eng.q8_linear(model.lm_head, eng.rmsnorm(last, model.final_norm, model.eps))


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16"])
def test_model_steps(oracle, kv_dtype):
    """A prompt and greedy steps of a model with normed heads, as its own entry points and as their parts.  Equal but
    for the rounding of the folded norms, which may move a K value over a code's border: 2e-2 of the logits' norm."""
    from test_gpu_model_q8 import _model
    model, _ = _model(oracle, 2, 4, 2, 512, 320, 5)
    for i, w in enumerate(model.layers):
        w.q_norm, w.k_norm = (1.5 + 0.2 * randn((128,), 70 + 2 * i + j) for j in range(2))
        w.q_norm, w.k_norm = w.q_norm.cuda(), w.k_norm.cuda()
    engines = [make_engine(4, 2, [64, 64], kv_dtype=kv_dtype, hidden=512, n_layers=2) for _ in range(2)]
    B, n_new, ids = 2, 24, [1, 0]
    tokens = torch.randint(0, 320, (B, n_new), generator=torch.Generator().manual_seed(1)).int().cuda()
    logits = torch.empty(B, 320, device="cuda")
    nxt = engines[0].prefill_step_q8(model, ids, tokens, logits=logits)
    want = _composed(engines[1], model, ids, tokens, n_new)
    for step in range(4):
        engines[0].sync()
        d = (logits - want).norm() / want.norm()
        assert d <= 2e-2, (step, float(d))
        assert [engines[0].seq_len(1, s) for s in (0, 1)] == [n_new + step] * 2
        want = _composed(engines[1], model, ids, nxt.clone(), 1)
        nxt = engines[0].decode_step_q8(model, ids, nxt, logits=logits)
    # the norms count: without them the same token's logits are others
    bare, norms = engines[0], [(w.q_norm, w.k_norm) for w in model.layers]
    for w in model.layers:
        w.q_norm = w.k_norm = None
    bare.reset()
    bare.prefill_step_q8(model, ids, tokens, logits=logits)
    engines[1].reset()
    for w, (a, b) in zip(model.layers, norms):
        w.q_norm, w.k_norm = a, b
    want = _composed(engines[1], model, ids, tokens, n_new)
    assert (logits - want).norm() > 0.1 * want.norm()
    for e in engines:
        e.close()
