"""The 4-bit cache where its arithmetic could run short of bits, each with a bound derived from its own roundings."""
import math

import numpy as np
import pytest
import torch

import q4_ref
from helpers import as_f32_np, make_engine, randn

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------- small weights
def _dominated(n, n_kv, seed):
    """Keys and values of n tokens: token 0's key is the dominant one and its value zero, the others' keys are equal and
    their values have a mean of 1, so that the output is what the small weights carry.  Constant groups are held as
    they are."""
    k = torch.zeros(n, n_kv, 128)
    k[0] = 1.546875  # against q = 1: 1.546875 * 128 / sqrt(128) = 17.501 nats = 2^25.25 times the others' weight
    v = (1 + 0.25 * randn((n, n_kv, 128), seed)).bfloat16().float()
    v[0] = 0
    return k, v


def _dominated_want(v, seen):
    w = math.exp(-1.546875 * 128 / math.sqrt(128))
    held = q4_ref.held(v).double()
    total = held[:seen].sum(0) * w  # token 0's value is zero
    return (total / (1 + (seen - 1) * w)).numpy()  # [n_kv, 128]


@pytest.mark.parametrize("heads", [(32, 8), (64, 8), (8, 1), (4, 1)])
@pytest.mark.parametrize("n,rows", [(300, 1), (8192, 128), (32768, 128)])
def test_decode_weights_below_a_dominant_key(heads, n, rows):
    """Weights are held as f16 pairs at 2^14 times their size: each is off by at most 2^-39 of the largest (half an f16
    subnormal step, scaled) besides its 22 bits, so an output by n * 2^-39 * max |v| and 1e-5 of its own size."""
    n_heads, n_kv = heads
    k, v = _dominated(n, n_kv, 3)
    eng = make_engine(n_heads, n_kv, [n], kv_dtype="q4")
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    q = torch.ones(rows, n_heads, 128, device="cuda")
    out, lse = eng.decode(0, [0] * rows, q, with_lse=True)
    eng.sync()
    want = np.repeat(_dominated_want(v, n), n_heads // n_kv, 0)
    err = np.abs(out.cpu().double().numpy() - want)
    assert (err <= n * 2.0 ** -39 * 2.5 + 1e-5 * np.abs(want)).all(), (err.max(), np.abs(want).max())
    want_lse = 1.546875 * 128 / math.sqrt(128) + math.log1p((n - 1) * math.exp(-1.546875 * 128 / math.sqrt(128)))
    np.testing.assert_allclose(lse.cpu().numpy(), want_lse, rtol=2e-6)
    eng.close()


@pytest.mark.parametrize("heads", [(28, 4), (16, 8)])
def test_prefill_weights_below_a_dominant_key(heads):
    """The expanded form's weights are f16 at 2^6 times their size: each is off by at most 2^-31 of the largest besides
    its 11 bits; the values are fp16 too."""
    n_heads, n_kv = heads
    n, n_new = 8192, 60
    k, v = _dominated(n, n_kv, 4)
    eng = make_engine(n_heads, n_kv, [n], kv_dtype="q4")
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    q = torch.ones(n_new, n_heads, 128, device="cuda", dtype=torch.bfloat16)
    out = eng.prefill(0, 0, q).cpu().double().numpy()
    eng.sync()
    for i in (0, n_new - 1):
        seen = n - n_new + i + 1
        want = np.repeat(_dominated_want(v, seen), n_heads // n_kv, 0)
        err = np.abs(out[i] - want)
        assert (err <= seen * 2.0 ** -31 * 2.5 + 2.0 ** -9 * np.abs(want)).all(), (err.max(), np.abs(want).max())
    eng.close()


@pytest.mark.parametrize("heads", [(4, 2), (16, 2)])
@pytest.mark.parametrize("qscale", [1e2, 1e3])
def test_scores_of_a_hundred_million(heads, qscale):
    """Keys at the edge of the format and large queries: scores (base 2) around 2^23 and 2^26.7, of which a unit in the
    last place is 1 and 8.  The running maximum is rounded up, so that no weight passes 2^14, whatever that rounding is,
    and f16 holds it: the greatest score takes all, as in 64 bits, where the next is a million behind.  What a value is
    then off by: decode, the weight's 22 bits on its offset and its code's share, |o| + |8 s| <= 3 max |v|, each; prefill,
    the 11 bits of the weight and of the value."""
    n_heads, n_kv = heads
    n, n_new = 500, 70
    k = (2e4 * randn((n, n_kv, 128), 1)).clamp(-59000, 59000)
    v = randn((n, n_kv, 128), 2, torch.bfloat16).float()
    eng = make_engine(n_heads, n_kv, [n], kv_dtype="q4")
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    kh, vh = q4_ref.held(k).transpose(0, 1).double(), q4_ref.held(v).transpose(0, 1).double()
    q = qscale * randn((n_new, n_heads, 128), 3, torch.bfloat16)
    lens = [n - n_new + i + 1 for i in range(n_new)]
    want, want_lse = q4_ref.attend(q, kh, vh, lens)
    # a score is off by 2^-20 (decode), or 2^-11 for the keys' own rounding, of sum |q_d k_d| / sqrt(128) at most: rows
    # whose two greatest scores lie twice that apart are one value's alone
    s = torch.einsum("thd,hld->thl", q.double(), kh.repeat_interleave(n_heads // n_kv, 0)) / 128 ** 0.5
    seen = torch.arange(n)[None, None] < torch.tensor(lens)[:, None, None]
    top = s.masked_fill(~seen, -math.inf).topk(2, -1).values
    size = (q.double().abs().sum(-1) * kh.abs().amax() / 128 ** 0.5).numpy()
    vmax = float(vh.abs().max())
    for form, got, lse in (("decode", *eng.decode(0, [0] * n_new, q.float().cuda(), lens=lens, with_lse=True)),
                           ("prefill", *eng.prefill(0, 0, q.cuda(), with_lse=True))):
        got, lse = got.cpu().double().numpy(), lse.cpu().double().numpy()
        off = 2.0 ** -20 if form == "decode" else 2.0 ** -11
        clear = (top[..., 0] - top[..., 1]).numpy() > 2 * off * size
        assert np.isfinite(got).all() and clear.mean() > 0.5, form
        bound = 6 * 2.0 ** -22 * vmax if form == "decode" else 2.0 ** -10 * np.abs(want) + 2.0 ** -22 * vmax
        assert (np.abs(got - want) <= bound)[clear].all(), form
        assert (np.abs(lse - want_lse) <= off * size).all(), form
    eng.sync()
    eng.close()


# ----------------------------------------------------------------------------------------------- the scale
def _held(x):
    """The definition that include/oomattn.h gives: the scale is the range times 1/15 in f32, rounded to bf16."""
    g = x.float().unflatten(-1, (4, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * (torch.ones(()) / 15)).bfloat16().half().float()
    o = (lo + 8 * s).half().float()
    c = torch.where(s > 0, ((g - o) / s).round().clamp(-8, 7), torch.zeros(()))
    return (o + c * s).flatten(-2)


def test_scale_on_a_border():
    """Groups whose (max - min) * (1/15) and (max - min) / 15 round to different bf16 numbers: the former is held, and
    what is held is within the format's bound of the row either way."""
    r = 1 + 3 * torch.rand(1 << 24, generator=torch.Generator().manual_seed(1))
    r = r[(r / 15).bfloat16() != (r * (torch.ones(()) / 15)).bfloat16()]
    n = r.numel() // 8
    assert n >= 8
    x = torch.rand(2 * n * 4, 32, generator=torch.Generator().manual_seed(2)) * r[:8 * n, None]
    x[:, 0], x[:, 31] = 0, r[:8 * n]
    k, v = x.view(2, n, 1, 128)
    eng = make_engine(4, 1, [n], kv_dtype="q4")
    eng.kv_write(0, 0, k.contiguous().cuda(), v.contiguous().cuda())
    kg, vg = eng.kv_gather(0, [0])
    eng.sync()
    np.testing.assert_array_equal(kg.cpu().numpy(), _held(k).numpy())
    np.testing.assert_array_equal(vg.cpu().numpy(), _held(v).numpy())
    assert ((kg.cpu().double() - k.double()).abs() <= q4_ref.code_bound(k)).all()
    eng.close()


# ----------------------------------------------------------------------------------------------- the prefill's two forms
def _filled(n_heads, n_kv, n, seed, cap):
    eng = make_engine(n_heads, n_kv, [cap], kv_dtype="q4", shuffle_seed=seed)
    for pool in eng.kv_pool():
        pool.fill_(0xFF)  # NaN in every slot that is not written
    k, v = (randn((n, n_kv, 128), seed + i, torch.bfloat16) for i in (1, 2))
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    return eng, q4_ref.held(k).transpose(0, 1).double(), q4_ref.held(v).transpose(0, 1).double()


def _by_rows(n_heads, n_kv, n_new, n):
    """Whether the queries run as decode rows (include/oomattn.h)."""
    most = 5 + 200000 // (n * n_kv) if n_heads // n_kv > 4 else 7 + 260000 // (n * n_kv)
    return n_new <= min(48, most)


def _expanded_bounds(q, k, v, seen):
    """want, lse and how far the expanded form's may be off, for one query [Hq, 128] that sees `seen` keys.
    K, V and the weights are rounded to 11 bits (2^-11 relative, q enters exactly): independent roundings c_i, of which
    the sum stays within 7 sqrt(sum c_i^2) but for one in 10^10 (Hoeffding).  A score's are 2^-11 |q_d k_d| scale, and
    reach the lse times w_j and the output times w_j (v - out).  The tensor core truncates a running sum once per 16
    keys by 2^-23 of it; f32 does the rest."""
    group = q.shape[0] // k.shape[0]
    kk, vv = (t[:, :seen].repeat_interleave(group, 0) for t in (k, v))
    scale, u = 1 / math.sqrt(128), 2.0 ** -11
    s = torch.einsum("hd,hld->hl", q, kk) * scale
    w = torch.softmax(s, -1)
    want, lse = torch.einsum("hl,hld->hd", w, vv), torch.logsumexp(s, -1)
    ds2 = torch.einsum("hd,hld->hl", q ** 2, kk ** 2) * (scale * u) ** 2
    dlse = 7 * torch.sqrt((w ** 2 * ds2).sum(-1)) + 1e-5 + ds2.amax(-1) * 7
    var = torch.einsum("hl,hld->hd", w ** 2 * ds2, (vv - want[:, None]) ** 2)
    var = var + 2 * u * u * torch.einsum("hl,hld->hd", w ** 2, vv ** 2)
    dout = 7 * torch.sqrt(var) + (seen * 2.0 ** -26 + ds2.amax() * 7) * vv.abs().amax()
    return want, lse, dout, dlse


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(28, 4), (8, 8), (10, 2), (9, 3), (8, 2), (16, 2)])
@pytest.mark.parametrize("n_new,prefix,rows", [(1, 0, True), (1, 50, True), (7, 9, True), (16, 100, True), (25, 111, True),
                                               (24, 1200, True), (60, 0, False), (100, 28, False), (300, 500, False),
                                               (60, 2000, False)])
def test_prefill_within_its_form(heads, n_new, prefix, rows, out_dtype):
    n = n_new + prefix
    assert _by_rows(*heads, n_new, n) == rows
    eng, k, v = _filled(*heads, n, 30, n + 100)
    q = randn((n_new, heads[0], 128), 33, torch.bfloat16)
    out, lse = eng.prefill(0, 0, q.cuda(), out_dtype=out_dtype, with_lse=True)
    eng.sync()
    out, lse = torch.from_numpy(as_f32_np(out)).double(), lse.cpu().double()
    half = 2.0 ** -8 if out_dtype == torch.bfloat16 else 0.0
    for i in sorted({*range(0, n_new, max(1, n_new // 16)), n_new - 1}):
        want, want_lse, dout, dlse = _expanded_bounds(q[i].double(), k, v, prefix + i + 1)
        if rows:  # q and p in 22 bits: the decode's bounds
            dout, dlse = torch.full_like(dout, 1.5e-4), 1e-5 + 2e-6 * want_lse.abs()
        err = (out[i] - want).abs() - half * want.abs()
        assert (err <= dout * (1 + half)).all(), (i, float(err.max()))
        assert ((lse[i] - want_lse).abs() <= dlse).all(), (i, float((lse[i] - want_lse).abs().max()))
        if rows and not half:
            assert (out[i] - want).norm() <= 1e-5 * want.norm()
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16"])
@pytest.mark.parametrize("n_new,prefix", [(20, 0), (100, 100), (64, 4000)])
def test_prefill_nan_key(n_new, prefix, kv_dtype):
    """A NaN of K reaches the queries that see its token, in out and lse both, and no other."""
    n, at = n_new + prefix, prefix + n_new // 2
    k, v = randn((n, 2, 128), 1), randn((n, 2, 128), 2)
    k[at, 1, 100] = math.nan
    eng = make_engine(8, 2, [n], kv_dtype=kv_dtype)
    eng.kv_write(0, 0, k.cuda(), v.cuda())
    q = randn((n_new, 8, 128), 3, torch.bfloat16)
    out, lse = eng.prefill(0, 0, q.cuda(), with_lse=True)
    eng.sync()
    sees = torch.arange(n_new) >= n_new // 2
    for x in (out.cpu().isnan().all(-1), out.cpu().isnan().any(-1), lse.cpu().isnan()):
        assert not x[:, :4].any() and torch.equal(x[:, 4:], sees[:, None].expand(-1, 4))
    eng.close()
