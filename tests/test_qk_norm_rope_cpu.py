"""Refusals of the query/key norm + rotation entry points (no GPU needed)."""

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
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


OVERLAP = 6


def c_call(t, views, d, dw=None):
    """The C entry's answer for operands at made-up addresses: ``views`` are
    (address, row stride, head stride, heads) of q, k, q_out, k_out, or with
    ``dw`` (two addresses) of q, k, dq, dk, dq_out, dk_out."""
    lib = _native.load()
    q, k, *rest = views
    if dw is None:
        order, fn = (q, rest[0], k, rest[1]), lib.bokt_qk_norm_rope
    else:
        order, fn = (q, rest[0], rest[2], k, rest[1], rest[3]), lib.bokt_qk_norm_rope_backward
    strides = (ctypes.c_int64 * 12)(*[x for v in order for x in v[1:3]])
    far = 1 << 50
    if dw is None:
        return fn(q[0], k[0], far, far, far, 0, far, 8, rest[0][0], rest[1][0], t, q[3], k[3], d, 2, strides, 0,
                  1e-6, 1, None)
    return fn(rest[2][0], rest[3][0], q[0], k[0], far, far, far, 0, far, 8, rest[0][0], rest[1][0], *dw, t, q[3],
              k[3], d, 2, strides, 0, 1e-6, 1, far, 1 << 40, None)


def bytes_of(t, view, d):
    p, row, head, h = view
    return {p + 2 * (i * row + j * head + e) + b for i in range(t) for j in range(h) for e in range(d) for b in (0, 1)}


def overlap_cases():
    """Layouts of real use that share no memory, then made-up ones of every kind
    against the bytes counted one by one."""
    t, h, hk, d = 5, 4, 2, 8
    base, n = 1 << 40, 2 * d
    packed = (h + 2 * hk) * d
    q, k = (base, packed, d, h), (base + n * h, packed, d, hk)
    apart = [
        (t, [q, k, q, k]),                                                    # in place in one projection output
        (t, [q, k, (base + (1 << 20), h * d, d, h), (base + (1 << 21), hk * d, d, hk)]),
        # outputs beside each other in one buffer; heads in front of tokens; q, k, v beside each other in every head
        (t, [q, k, (base + (1 << 20), (h + hk) * d, d, h), (base + (1 << 20) + n * h, (h + hk) * d, d, hk)]),
        (t, [(base, d, t * d, h), (base + n * h * t, d, t * d, hk)] * 2),
        (t, [(base, 3 * h * d, 3 * d, h), (base + n, 3 * h * d, 3 * d, h)] * 2),
        (t, [(base, 3 * d, 3 * t * d, h), (base + n, 3 * d, 3 * t * d, h)] * 2),
        (t, [(base, 0, 0, h), (base, 0, 0, h), (base + (1 << 20), h * d, d, h), (base + (1 << 21), h * d, d, h)]),
        (1, [(base, 7, d, h), (base + n * h, 999, d, hk)] * 2),               # one token: any row stride
        (t, [(base, packed, d, h), (base + n * h, packed, 12345, 1)] * 2),    # one key head: any head stride
        (t, [q, (base, packed, d, 0), q, (base, packed, d, 0)]),
        (0, [q, q, q, q]),
    ]
    for t_, views in apart:
        assert c_call(t_, views, d) != OVERLAP, views
        grads = [(v[0] + (1 << 30), *v[1:]) for v in views[2:]]
        for extra in (grads, views[2:], views[:2]):
            assert c_call(t_, views + extra, d, (1 << 45, (1 << 45) + 4 * d)) != OVERLAP, views
    rng = np.random.default_rng(0)
    hit = told = 0
    for _ in range(3000):
        t, d = int(rng.integers(1, 5)), int(rng.integers(2, 5))
        hs = [int(rng.integers(0, 4)) for _ in range(2)]

        def view(h, free):
            head = int(rng.integers(0 if free else d, 3 * d))
            row = int(rng.choice([max(h, 1) * head, 3 * d * max(h, 1), int(rng.integers(0, 40))]))
            return (base + 2 * int(rng.integers(0, 160)), row, head, h)

        views = [view(h, True) for h in hs] + [view(h, False) for h in hs]
        if rng.random() < 0.3:
            views[2] = views[0]
        if rng.random() < 0.3:
            views[3] = views[1]
        at = [bytes_of(t, v, d) for v in views]
        true = bool(at[2] & at[3]) or bool(at[2] & at[1]) or bool(at[3] & at[0]) or \
            (views[2] != views[0] and bool(at[2] & at[0])) or (views[3] != views[1] and bool(at[3] & at[1]))
        rc = c_call(t, views, d)
        # Two views that differ only in strides that nothing takes are the same view.
        unused = [(v[0], 0 if t == 1 else v[1], 0 if v[3] <= 1 else v[2], v[3]) for v in views]
        same = unused[2] == unused[0] and views[2] != views[0] or unused[3] == unused[1] and views[3] != views[1]
        if true and not same:
            assert rc == OVERLAP, (t, d, views)
            hit += 1
        told += rc == OVERLAP and not true
    # Refused without an overlap: only interleavings that no common stride explains.
    assert hit > 1000 and told < 500, (hit, told)
    # The gradients' own operands.
    t, d = 3, 8
    q, k, dq, dk, go, gk = [(base + (i << 12), h * d, d, h) for i, h in enumerate((4, 2, 4, 2, 4, 2))]
    dw = (base + (9 << 12), base + (10 << 12))
    assert c_call(t, [q, k, dq, dk, go, gk], d, dw) != OVERLAP
    for bad in ([q, k, dq, dk, (dq[0] + 16, *dq[1:]), gk], [q, k, dq, dk, dk[:3] + (4,), gk],
                [q, k, dq, dk, go, (dq[0], *gk[1:])], [q, k, gk[:3] + (4,), dk, go, gk], [q, k, dq, dq[:3] + (2,), go, gk]):
        assert c_call(t, bad, d, dw) == OVERLAP, bad
    for bad in ((dq[0], dw[1]), (dw[0], dk[0] + 2 * 3 * 2 * 8 - 4), (dw[0], dw[0] + 4 * d - 4)):
        assert c_call(t, [q, k, dq, dk, go, gk], d, bad) == OVERLAP, bad
    assert b"dq_weight must not overlap dk_weight" in _native.load().bokt_last_error()


def test_overlapping_operands_are_refused():
    """In a process without a device, where nothing can be launched on the
    addresses, whatever the answer."""
    root = Path(__file__).resolve().parents[1]
    code = "from tests.test_qk_norm_rope_cpu import overlap_cases; overlap_cases(); print('done')"
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]


def test_overlap_is_a_value_error():
    with pytest.raises(ValueError, match="overlapping memory"):
        _native.check(OVERLAP, "call")
