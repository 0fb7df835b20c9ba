"""Refusals of the adapter bank and the projection with adapters (no GPU needed)."""

import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import lora_gemm

BF = torch.bfloat16


def bank(**over):
    return lora_gemm.AdapterBank(**{**dict(slots=4, k=16, n=24, max_rank=8, dtype=BF, device="cpu"), **over})


@pytest.mark.parametrize("over, match", [
    (dict(slots=0), "slots"), (dict(slots=1025), "slots"), (dict(k=12), "multiples of 8"),
    (dict(n=0), "multiples of 8"), (dict(max_rank=0), "max_rank"), (dict(max_rank=129), "max_rank"),
    (dict(dtype=torch.float32), "dtype"),
])
def test_bank_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        bank(**over)


def test_bank_load_and_unload():
    b = bank()
    assert b.rank == 16
    a1, b1 = torch.randn(8, 16).to(BF), torch.randn(8, 24).to(BF)
    b.load(2, a1, b1, 0.5)
    assert torch.equal(b.a[2, :8], a1) and torch.equal(b.b[2, :8], b1)
    assert not b.a[2, 8:].any() and b.ranks.tolist() == [0, 0, 8, 0] and b.scales[2] == 0.5
    b.load(2, a1[:3], b1[:3])  # a smaller adapter leaves nothing of the larger one
    assert not b.a[2, 3:].any() and not b.b[2, 3:].any() and b.ranks[2] == 3
    b.unload(2)
    assert not b.a.any() and not b.b.any() and not b.ranks.any() and not b.scales.any()


@pytest.mark.parametrize("args, match", [
    ((4, (8, 16), (8, 24)), "slot"), ((-1, (8, 16), (8, 24)), "slot"),
    ((0, (9, 16), (9, 24)), "shape mismatch"), ((0, (0, 16), (0, 24)), "shape mismatch"),
    ((0, (8, 24), (8, 24)), "shape mismatch"), ((0, (8, 16), (7, 24)), "shape mismatch"),
])
def test_load_refusals(args, match):
    slot, a, b = args
    with pytest.raises(ValueError, match=match):
        bank().load(slot, torch.zeros(a, dtype=BF), torch.zeros(b, dtype=BF))


def test_load_refuses_types_and_values_that_are_not_finite():
    b, a1, b1 = bank(), torch.zeros(4, 16, dtype=BF), torch.zeros(4, 24, dtype=BF)
    with pytest.raises(ValueError, match="dtype"):
        b.load(0, a1.half(), b1)
    for scale in (float("inf"), float("nan"), 1e39):
        with pytest.raises(ValueError, match="scale"):
            b.load(0, a1, b1, scale)
    for bad in (float("inf"), float("nan")):
        x = b1.clone()
        x[3, 7] = bad
        with pytest.raises(ValueError, match="finite"):
            b.load(0, a1, x)
        x = a1.clone()
        x[0, 0] = bad
        with pytest.raises(ValueError, match="finite"):
            b.load(0, x, b1)
    assert not b.ranks.any()


def call(t=3, **over):
    a = {"x": torch.zeros(t, 16, dtype=BF), "w": torch.zeros(16, 24, dtype=BF), "bank": bank(),
         "ids": torch.zeros(t, dtype=torch.int32), "out": torch.zeros(t, 24, dtype=BF)}
    return lora_gemm.launch(**{**a, **over})


@pytest.mark.parametrize("over, match", [
    (dict(w=torch.zeros(24, 24, dtype=BF)), "shape mismatch"),
    (dict(out=torch.zeros(4, 24, dtype=BF)), "shape mismatch"),
    (dict(bank=bank(n=32)), "bank"),
    (dict(ids=torch.zeros(4, dtype=torch.int32)), "ids"),
    (dict(ids=torch.zeros(3, dtype=torch.int64)), "ids"),
    (dict(ids=torch.zeros(6, dtype=torch.int32)[::2]), "ids"),
    (dict(bank=bank(dtype=torch.float16)), "share one dtype"),
    (dict(x=torch.zeros(16, 3, dtype=BF).t()), "contiguous"),
    ({}, "CUDA"),
])
def test_launch_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        call(**over)


def test_bank_loads_what_other_memory_holds():
    """Strided and transposed adapters are copied, not referenced."""
    b = bank()
    a1, b1 = torch.randn(16, 8).to(BF), torch.randn(8, 48).to(BF)
    b.load(1, a1.t(), b1[:, ::2], 2.0)
    want = a1.t().clone()
    a1.zero_()
    assert torch.equal(b.a[1, :8], want) and torch.equal(b.b[1, :8], b1[:, ::2])


def test_c_abi_argument_errors_need_no_gpu():
    lib = _native.load()

    def rc(m=1, n=8, k=8, slots=1, rank=16, dtype=1):
        return lib.bokt_lora_gemm(*[None] * 8, m, n, k, slots, rank, dtype, None, 0, None)

    assert rc(dtype=2) == 1 and b"dtype" in lib.bokt_last_error()
    assert rc(m=-1) == 1 and rc(n=0) == 1 and rc(slots=0) == 1 and rc(rank=24) == 1
    assert rc(slots=1025) == 2 and rc(k=12) == 2 and rc(n=4) == 2
    assert rc(m=0) == 0
    assert rc() == 1 and b"null" in lib.bokt_last_error()


def test_sizes_past_32_bits_are_refused():
    lib, most = _native.load(), 1 << 30
    for sizes in ((most + 1, 24, 16), (8, most + 8, 16), (8, 24, most + 8)):
        assert lib.bokt_lora_gemm_workspace_bytes(*sizes, 4, 16) == -1
    null = [None] * 8
    assert lib.bokt_lora_gemm(*null, most + 1, 24, 16, 4, 16, _native.BF16, None, 0, None) != 0
    assert b"2^30" in lib.bokt_last_error()
    b = bank()
    x, w, ids = torch.zeros(1, 16, dtype=BF), torch.zeros(16, 24, dtype=BF), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        lora_gemm.launch(x.expand(most + 1, 16), w, b, ids, torch.zeros(1, 24, dtype=BF).expand(most + 1, 24))


@pytest.mark.parametrize("scale, size, e", [
    (1.0, 1.5, 0), (0.5, 0.6, 1), (1e6, 2e-3, 9), (-4.0, 6e-8, 24), (1.0, 3e4, 0), (0.3, 3.0, -1), (1e-6, 3.0, -1),
    (1e-6, 3e4, -14), (2.0**-3, 3e4, -3), (0.0, 3e4, 0), (1.0, 0.0, 0),
])
def test_fp16_slots_move_a_power_of_two_from_the_scale(scale, size, e):
    """The product of scale and b is kept, the larger ones of b exactly."""
    bk = bank(dtype=torch.float16)
    a1, b1 = torch.randn(4, 16).half(), (torch.rand(4, 24) * size / 2).half()
    b1[2, 5] = -size
    bk.load(1, a1, b1, scale)
    assert torch.equal(bk.b[1, :4].double(), (b1 * 2.0**e).half().double())
    assert bk.scales[1] == torch.tensor(scale * 2.0**-e, dtype=torch.float32)
    assert torch.equal(bk.a[1, :4], a1) and bk.ranks[1] == 4
    if e >= 0:
        assert torch.equal(bk.b[1, :4].double() * 2.0**-e, b1.double())


def test_parameters_loaded_into_the_bank_leave_no_graph():
    """A bank is storage: loading trained parameters records no history on it."""
    b = bank()
    a1 = torch.nn.Parameter(torch.randn(8, 16).to(BF))
    b1 = torch.nn.Parameter(torch.randn(8, 24).to(BF))
    b.load(0, a1, b1)
    b.load(0, a1[:3], b1[:3])
    for t in (b.a, b.b, b.scales, b.ranks):
        assert not t.requires_grad and t.grad_fn is None
    b.unload(0)
    b.load(0, a1[:3], b1[:3])
    assert torch.equal(b.a[0, :3], a1[:3]) and not b.a[0, 3:].any()


def test_fp16_parameters_leave_no_graph_either():
    b = bank(dtype=torch.float16)
    a1, b1 = torch.nn.Parameter(torch.randn(8, 16).half()), torch.nn.Parameter(torch.full((8, 24), 0.25).half())
    b.load(0, a1, b1, 1e5)
    assert not (b.a.requires_grad or b.b.requires_grad or b.scales.requires_grad) and b.b[0, 0, 0] == 1


def test_other_numbers_of_dimensions_are_refused():
    for shape in ((), (16,), (1, 16, 1)):
        with pytest.raises(ValueError, match="shape mismatch"):
            bank().load(0, torch.zeros(shape, dtype=BF), torch.zeros(1, 24, dtype=BF))
    for over in (dict(w=torch.zeros(16, dtype=BF)), dict(x=torch.zeros(16, dtype=BF)), dict(x=torch.zeros(3, 1, 16, dtype=BF))):
        with pytest.raises(ValueError, match="dimensions"):
            call(**over)
