"""RMSNorm of every query and key head and the rotary rotation in one pass (sm_100a).

The step between a decoder layer's query/key projection and its attention:
the RMSNorm of the reference's ``bo_kernel_tuner/kernels/rmsnorm.py:22-25``
over each head (size D), ``y = x * rsqrt(mean(x^2) + epsilon) * w``, followed
by the position rotation of ``y[:rot]`` (the reference has no rotation), in
fp32 with one rounding.  ``launch`` is the forward pass, ``launch_backward``
its gradients; neither allocates anything a caller sees, both can be captured
in a CUDA graph.

``q`` [T, H, D] and ``k`` [T, Hk, D] may be views into the projection's output
(any strides, last dimension contiguous); ``positions`` is int32 or int64 [T];
``cos_sin`` fp32 [P, rot] holds rot / 2 cosines and then rot / 2 sines per
position (``rope_table``).  A position outside [0, P) sets the device status
word (``_native.device_status``) and leaves that token's rows unwritten.

The rotation turns the pairs (i, i + rot / 2), or with ``interleaved`` the
neighbours (2 i, 2 i + 1).
"""

import math
import struct

from flashattentionanycard_b200 import _native

MAX_HEAD_ROWS = (1 << 31) - (1 << 16)


def rope_table(rows, rot, base=10000.0, device="cuda"):
    """fp32 [rows, rot]: cosines and sines of p * base^(-2 i / rot), angles in 64 bits."""
    import torch

    rows, rot = int(rows), int(rot)
    if not 0 <= rows < 1 << 31 or not 2 <= rot < 1 << 31 or rot % 2:
        raise ValueError("rows must be non-negative, rot even and positive, both below 2^31")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be finite and positive")
    out = torch.empty((rows, rot), device=device, dtype=torch.float32)
    with torch.cuda.device(out.device):
        _native.check(
            _native.load().bokt_rope_table(out.data_ptr(), rows, rot, float(base),
                                           _native.current_stream(out.device)),
            "bokt_rope_table",
        )
    return out


# Decode calls are shorter than their checks: each check below is a plain
# comparison, and every attribute is read once.
_pack8, _pack12 = struct.Struct("8q").pack, struct.Struct("12q").pack  # int64 strides


def _views(named, shape, dtype, index):
    """Checks views of one shape, (name, view, written) each; returns their row
    and head strides in order."""
    n, h, d = shape
    out = []
    for name, x, written in named:
        if x.shape != shape:
            raise ValueError(f"shape mismatch: {name} {tuple(x.shape)}, expected {tuple(shape)}")
        if x.dtype != dtype:
            raise ValueError(f"{name} must share q's dtype")
        row, head, last = x.stride()
        if last != 1 and d > 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        # Distinct elements of an output must be distinct memory.
        if written and not (
                (head >= d and row >= head * (h - 1) + d) or (row >= d and head >= row * (n - 1) + d)
                or n * h <= 1 or (n == 1 and head >= d) or (h == 1 and row >= d)):
            raise ValueError(f"{name} must not overlap itself (strides {x.stride()})")
        if x.get_device() != index:
            raise ValueError("all tensors must be on one CUDA device")
        out += (row, head)
    return out


def _weight(name, w, d, dtype, index):
    if w.shape != (d,) or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {d} elements")
    if w.dtype != dtype:
        raise ValueError(f"{name} must " + ("be fp32" if name.startswith("d") else "share q's dtype"))
    if w.get_device() != index:
        raise ValueError("all tensors must be on one CUDA device")


def _check(q, k, q_weight, k_weight, positions, cos_sin, epsilon):
    """(q's shape, k's shape, rot, device index, is int64) of a call; checks all
    that both directions share except the views."""
    import torch

    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3:
        raise ValueError(f"q and k must be [tokens, heads, head size], got {tuple(qs)} and {tuple(ks)}")
    t, h, d = qs
    if ks[0] != t or ks[2] != d:
        raise ValueError(f"shape mismatch: q {tuple(qs)}, k {tuple(ks)}")
    if t * (h + ks[1]) > MAX_HEAD_ROWS or t > MAX_HEAD_ROWS:
        raise ValueError(f"at most {MAX_HEAD_ROWS} head rows (got {t} tokens of {h} + {ks[1]} heads)")
    index = q.get_device()
    _weight("q_weight", q_weight, d, q.dtype, index)
    _weight("k_weight", k_weight, d, q.dtype, index)
    i64 = positions.dtype == torch.int64
    if not (i64 or positions.dtype == torch.int32) or positions.shape != (t,) or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor of {t} elements")
    table = cos_sin.shape
    if cos_sin.dtype != torch.float32 or len(table) != 2 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous fp32 [positions, rot] tensor")
    rot = table[1]
    if table[0] > MAX_HEAD_ROWS:
        raise ValueError(f"cos_sin must have at most {MAX_HEAD_ROWS} rows, got {table[0]}")
    if rot < 2 or rot % 2 or rot > d:
        raise ValueError(f"rot (cos_sin's width) must be even and in [2, {d}], got {rot}")
    if not (epsilon >= 0 and math.isfinite(epsilon)):
        raise ValueError("epsilon must be finite and non-negative")
    if positions.get_device() != index or cos_sin.get_device() != index:
        raise ValueError("all tensors must be on one CUDA device")
    return qs, ks, rot, table[0], index, 1 if i64 else 0


def launch(q, k, q_weight, k_weight, positions, cos_sin, q_out, k_out, epsilon=1e-6, interleaved=False):
    """q_out, k_out = rotated norms of q's and k's heads (q_out may be q, k_out
    may be k; outputs that overlap otherwise are a ValueError)."""
    import torch

    qs, ks, rot, rows, index, i64 = _check(q, k, q_weight, k_weight, positions, cos_sin, epsilon)
    dtype = q.dtype
    strides = _pack8(*_views((("q", q, False), ("q_out", q_out, True)), qs, dtype, index),
                     *_views((("k", k, False), ("k_out", k_out, True)), ks, dtype, index))
    if index < 0:
        raise ValueError("q, k and their tensors must be CUDA tensors")
    if torch._C._cuda_getDevice() != index:  # the library launches on the current device
        with torch.cuda.device(index):
            return launch(q, k, q_weight, k_weight, positions, cos_sin, q_out, k_out, epsilon, interleaved)
    rc = _native.load().bokt_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(), i64,
        cos_sin.data_ptr(), rows, q_out.data_ptr(), k_out.data_ptr(), qs[0], qs[1], ks[1], qs[2], rot,
        strides, 1 if interleaved else 0, epsilon, _native.dtype_code(dtype),
        torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, "bokt_qk_norm_rope")
    return q_out, k_out


def launch_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, cos_sin, dq, dk, dq_weight,
                    dk_weight, epsilon=1e-6, interleaved=False):
    """Gradients of ``launch``: dq, dk (q's dtype; dq may be dq_out or q, dk may
    be dk_out or k; any other overlap is a ValueError) and dq_weight, dk_weight
    (fp32 [D], overwritten, summed in a fixed order: the same inputs give the
    same bits)."""
    import torch

    qs, ks, rot, rows, index, i64 = _check(q, k, q_weight, k_weight, positions, cos_sin, epsilon)
    dtype, d = q.dtype, qs[2]
    strides = _pack12(
        *_views((("q", q, False), ("dq", dq, True), ("dq_out", dq_out, False)), qs, dtype, index),
        *_views((("k", k, False), ("dk", dk, True), ("dk_out", dk_out, False)), ks, dtype, index))
    _weight("dq_weight", dq_weight, d, torch.float32, index)
    _weight("dk_weight", dk_weight, d, torch.float32, index)
    if abs(dq_weight.data_ptr() - dk_weight.data_ptr()) < 4 * d:
        raise ValueError("dq_weight and dk_weight must be separate buffers (add them where q and k share a weight)")
    if index < 0:
        raise ValueError("q, k and their tensors must be CUDA tensors")
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return launch_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, cos_sin, dq, dk,
                                   dq_weight, dk_weight, epsilon, interleaved)
    scratch, nbytes = _native.workspace("bokt_qk_norm_rope_workspace_bytes", (d,), index, None)
    rc = _native.load().bokt_qk_norm_rope_backward(
        dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), q_weight.data_ptr(),
        k_weight.data_ptr(), positions.data_ptr(), i64, cos_sin.data_ptr(), rows, dq.data_ptr(),
        dk.data_ptr(), dq_weight.data_ptr(), dk_weight.data_ptr(), qs[0], qs[1], ks[1], d, rot, strides,
        1 if interleaved else 0, epsilon, _native.dtype_code(dtype), scratch.data_ptr(), nbytes,
        torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, "bokt_qk_norm_rope_backward")
    return dq, dk, dq_weight, dk_weight
