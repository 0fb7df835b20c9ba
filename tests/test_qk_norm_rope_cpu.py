"""Refusals of the query/key norm + rotation entry points (no GPU needed)."""

import ctypes

import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import qk_norm_rope


def call(t=3, h=2, hk=1, d=16, rot=16, backward=False, **over):
    bf = torch.bfloat16
    a = {"q": torch.zeros(t, h, d, dtype=bf), "k": torch.zeros(t, hk, d, dtype=bf),
         "q_weight": torch.zeros(d, dtype=bf), "k_weight": torch.zeros(d, dtype=bf),
         "positions": torch.zeros(t, dtype=torch.int32), "cos_sin": torch.zeros(4, rot)}
    outs = {"q_out": torch.zeros(t, h, d, dtype=bf), "k_out": torch.zeros(t, hk, d, dtype=bf)}
    if backward:
        outs = {"dq": outs["q_out"], "dk": outs["k_out"], "dq_out": torch.zeros(t, h, d, dtype=bf),
                "dk_out": torch.zeros(t, hk, d, dtype=bf), "dq_weight": torch.zeros(d),
                "dk_weight": torch.zeros(d)}
    fn = qk_norm_rope.launch_backward if backward else qk_norm_rope.launch
    fn(**{**a, **outs, **over})


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over, match", [
    (dict(q=torch.zeros(3, 16, dtype=torch.bfloat16)), "heads, head size"),
    (dict(k=torch.zeros(4, 1, 16, dtype=torch.bfloat16)), "shape mismatch"),
    (dict(k=torch.zeros(3, 1, 8, dtype=torch.bfloat16)), "shape mismatch"),
    (dict(k=torch.zeros(3, 1, 16, dtype=torch.float16)), "share q's dtype"),
    (dict(q_weight=torch.zeros(8, dtype=torch.bfloat16)), "q_weight"),
    (dict(k_weight=torch.zeros(16)), "share q's dtype"),
    (dict(positions=torch.zeros(3)), "positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions"),
    (dict(cos_sin=torch.zeros(4, 16, dtype=torch.float64)), "cos_sin"),
    (dict(cos_sin=torch.zeros(4, 15)), "rot"),
    (dict(cos_sin=torch.zeros(4, 18)), "rot"),
    (dict(cos_sin=torch.zeros(4, 0)), "rot"),
    (dict(epsilon=float("nan")), "epsilon"),
    (dict(epsilon=-1.0), "epsilon"),
    (dict(q=torch.zeros(3, 2, 32, dtype=torch.bfloat16)[..., ::2]), "last dimension"),
    ({}, "CUDA"),
])
def test_refusals(over, match, backward):
    with pytest.raises(ValueError, match=match):
        call(backward=backward, **over)


@pytest.mark.parametrize("name, backward", [("q_out", False), ("dq", True)])
def test_outputs_that_overlap_themselves_are_refused(name, backward):
    for view in (torch.zeros(1, 1, 16, dtype=torch.bfloat16).expand(3, 2, 16),
                 torch.zeros(200, dtype=torch.bfloat16).as_strided((3, 2, 16), (24, 16, 1)),
                 torch.zeros(200, dtype=torch.bfloat16).as_strided((3, 2, 16), (16, 8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            call(backward=backward, **{name: view})


def test_gradient_buffers_of_weights_are_fp32():
    with pytest.raises(ValueError, match="fp32"):
        lib_free = torch.zeros(16, dtype=torch.bfloat16)
        call(backward=True, dq_weight=lib_free)


def test_rope_table_refusals():
    for bad in (dict(rows=-1, rot=4), dict(rows=4, rot=3), dict(rows=4, rot=0),
                dict(rows=4, rot=4, base=0.0), dict(rows=4, rot=4, base=float("inf"))):
        with pytest.raises(ValueError):
            qk_norm_rope.rope_table(**bad, device="cpu")


def test_c_abi_argument_errors_need_no_gpu():
    lib = _native.load()
    st = (ctypes.c_int64 * 8)()
    args = lambda **o: [None] * 5 + [0, None, 0, None, None] + [  # noqa: E731
        o.get("t", 1), 1, 1, o.get("d", 16), o.get("rot", 16), st, 0, o.get("eps", 1e-6), o.get("dtype", 1), None]
    assert lib.bokt_qk_norm_rope(*args(dtype=2)) == 1 and b"dtype" in lib.bokt_last_error()
    assert lib.bokt_qk_norm_rope(*args(t=-1)) == 1
    assert lib.bokt_qk_norm_rope(*args(d=2000)) == 2
    assert lib.bokt_qk_norm_rope(*args(rot=15)) == 1
    assert lib.bokt_qk_norm_rope(*args(eps=float("nan"))) == 1
    assert lib.bokt_rope_table(None, 4, 3, 10000.0, None) == 1
    assert lib.bokt_rope_table(None, 0, 4, 10000.0, None) == 0


def test_one_buffer_for_both_weight_gradients_is_refused():
    both = torch.zeros(16)
    with pytest.raises(ValueError, match="separate"):
        call(backward=True, dq_weight=both, dk_weight=both)


@pytest.mark.parametrize("backward", [False, True])
def test_sizes_past_32_bits_are_refused(backward):
    bf = torch.bfloat16
    many = torch.zeros(1, 1, 16, dtype=bf).expand(3, 1 << 30, 16)
    with pytest.raises(ValueError, match="head rows"):
        call(backward=backward, q=many)
    with pytest.raises(ValueError, match="head rows"):
        call(backward=backward, k=many)
    none = torch.zeros(1, 0, 16, dtype=bf).expand(1 << 32, 0, 16)
    with pytest.raises(ValueError, match="head rows"):
        call(backward=backward, q=none, k=none)
    with pytest.raises(ValueError, match="2\\^31"):
        qk_norm_rope.rope_table(1 << 31, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        qk_norm_rope.rope_table(4, 1 << 31)
