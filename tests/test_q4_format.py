"""The error bound that include/oomattn.h states for a value in the 4-bit cache, on the restatement of the format."""
import math

import pytest
import torch

import q4_ref


def _bound(x):
    _, s, o = q4_ref.quantize(x)
    return (0.53 * s + 2.0 ** -11 * o.abs() + 5e-7).double().repeat_interleave(32, -1)


def _rows(kind):
    g = torch.Generator().manual_seed(len(kind))
    r = torch.rand(4000, 128, generator=g)
    n = torch.randn(4000, 128, generator=g)
    m = torch.exp2(24 * torch.rand(4000, 1, generator=g) - 9)  # sizes from 2^-9 to 2^15
    return {"normal": n, "uniform": r, "sizes": (n * m).clamp(-60000, 60000), "shifted": n + 300 * r[:, :1],
            "narrow": 500 + 1000 * r[:, :1] + 1e-3 * n, "tiny": 15 * 1.4 * 2.0 ** -24 * r, "tinier": 3e-7 * r + 1e-3 * n[:, :1],
            "outliers": n + 200 * (r > 0.99), "constant": (n * m)[:, :1].clamp(-60000, 60000).expand(-1, 128)}[kind]


@pytest.mark.parametrize("kind", ["normal", "uniform", "sizes", "shifted", "narrow", "tiny", "tinier", "outliers", "constant"])
def test_values_are_within_the_stated_bound(kind):
    x = _rows(kind).contiguous()
    err = (q4_ref.held(x).double() - x.double()).abs()
    assert (err <= _bound(x)).all(), float((err / _bound(x)).max())


def test_the_examples_of_the_bound():
    x = torch.full((1, 128), 513.25)
    assert float((q4_ref.held(x) - x).abs().max()) == 0.25 == 2.0 ** -11 * 512  # a half-precision offset's half step
    # a range that the scale cannot hold: the least value is what remains
    x = 0.25 + 2.0 ** -25 * torch.arange(128)[None] / 32
    assert (q4_ref.held(x) == 0.25).all()
    assert math.isnan(float(q4_ref.held(torch.where(torch.arange(128) == 3, math.nan, x))[0, 5]))
