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
