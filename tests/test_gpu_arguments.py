"""Counts, places and sizes of a call's arguments that do not fit one another: refused before anything is read."""
import pytest
import torch

from helpers import make_engine

pytestmark = pytest.mark.gpu


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
