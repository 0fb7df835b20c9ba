"""Refusals of the few-token MoE layer (no GPU needed)."""

import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import moe_decode

BF = torch.bfloat16


def call(t=3, e=4, k=16, inner=8, topk=2, **over):
    a = {"x": torch.zeros(t, k, dtype=BF), "logits": torch.zeros(t, e),
         "w_gate_up": torch.zeros(e, k, 2 * inner, dtype=BF), "w_down": torch.zeros(e, inner, k, dtype=BF),
         "out": torch.zeros(t, k, dtype=BF), "topk": topk}
    return moe_decode.launch(**{**a, **over})


@pytest.mark.parametrize("kw, match", [
    (dict(x=torch.zeros(3, 1, 16, dtype=BF)), "dimensions"),
    (dict(x=torch.zeros(3, 24, dtype=BF)), "shape mismatch"),
    (dict(w_gate_up=torch.zeros(4, 16, 24, dtype=BF)), "shape mismatch"),
    (dict(w_down=torch.zeros(4, 8, 24, dtype=BF)), "shape mismatch"),
    (dict(logits=torch.zeros(3, 5)), "logits"),
    (dict(out=torch.zeros(4, 16, dtype=BF)), "out"),
    (dict(topk=0), "topk"),
    (dict(topk=5), "topk"),
    (dict(e=16, topk=9), "topk"),
    (dict(t=129), "at most 128"),
    (dict(e=1025), "1024"),
    (dict(k=20), "multiples of 8"),
    (dict(inner=12), "multiples of 8"),
    (dict(out=torch.zeros(3, 16)), "share one dtype"),
    (dict(logits=torch.zeros(3, 4, dtype=torch.float64)), "dtype"),
    (dict(x=torch.zeros(16, 3, dtype=BF).t()), "contiguous"),
    (dict(), "CUDA"),
])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


def test_c_abi_argument_errors_need_no_gpu():
    lib = _native.load()

    def rc(t=1, e=4, k=16, i=8, topk=2, logits=2, dtype=1):
        return lib.bokt_moe_decode(None, None, logits, None, None, None, t, e, k, i, topk, 1, dtype, None, 0, None)

    assert rc(dtype=2) == 1 and b"dtype" in lib.bokt_last_error()
    assert rc(logits=7) == 1
    assert rc(t=-1) == 1 and rc(e=0) == 1 and rc(topk=0) == 1 and rc(topk=5) == 1
    assert rc(t=129) == 2 and rc(e=2000, topk=1) == 2 and rc(e=16, topk=9) == 2
    assert rc(k=12) == 2 and rc(i=4) == 2 and rc(k=65544) == 2
    assert rc(t=0) == 0
    assert rc() == 1 and b"null" in lib.bokt_last_error()
