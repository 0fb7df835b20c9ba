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

import ctypes
import math

from flashattentionanycard_b200 import _native


def rope_table(rows, rot, base=10000.0, device="cuda"):
    """fp32 [rows, rot]: cosines and sines of p * base^(-2 i / rot), angles in 64 bits."""
    import torch

    rows, rot = int(rows), int(rot)
    if rows < 0 or rot < 2 or rot % 2:
        raise ValueError("rows must be non-negative and rot even and positive")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be finite and positive")
    out = torch.empty((rows, rot), device=device, dtype=torch.float32)
    with _native.on_device(out.device):
        _native.check(
            _native.load().bokt_rope_table(out.data_ptr(), rows, rot, float(base),
                                           _native.current_stream(out.device)),
            "bokt_rope_table",
        )
    return out


def _check(named, q, k, positions, cos_sin, weights, epsilon, writes):
    """Shapes, types, layouts and devices of a call; returns (tokens, head size, rot).

    Decode calls are shorter than these checks, so each is a plain comparison."""
    import torch

    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [tokens, heads, head size], got {tuple(q.shape)} and {tuple(k.shape)}")
    t, _, d = q.shape
    if k.shape[0] != t or k.shape[2] != d:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}")
    dtype, device = q.dtype, q.device
    for name, x, like in named:
        if x.shape != like.shape:
            raise ValueError(f"shape mismatch: {name} {tuple(x.shape)}, expected {tuple(like.shape)}")
        if x.dtype != dtype:
            raise ValueError(f"{name} must share q's dtype")
        row, head, last = x.stride()
        if last != 1 and d > 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        if name in writes:
            # Distinct elements of an output must be distinct memory.
            n, h, _ = x.shape
            if not (n * h <= 1 or (n == 1 and head >= d) or (h == 1 and row >= d)
                    or (head >= d and row >= head * (h - 1) + d) or (row >= d and head >= row * (n - 1) + d)):
                raise ValueError(f"{name} must not overlap itself (strides {x.stride()})")
    for name, w, wtype in weights:
        if w.shape != (d,) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of {d} elements")
        if w.dtype != (wtype or dtype):
            raise ValueError(f"{name} must " + ("be fp32" if wtype else "share q's dtype"))
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (t,) \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor of {t} elements")
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous fp32 [positions, rot] tensor")
    rot = cos_sin.shape[1]
    if rot < 2 or rot % 2 or rot > d:
        raise ValueError(f"rot (cos_sin's width) must be even and in [2, {d}], got {rot}")
    if not (math.isfinite(epsilon) and epsilon >= 0):
        raise ValueError("epsilon must be finite and non-negative")
    if not (q.is_cuda and positions.device == device and cos_sin.device == device
            and all(x.device == device for _, x, _ in named) and all(w.device == device for _, w, _ in weights)):
        raise ValueError("all tensors must be on one CUDA device")
    return t, d, rot


def launch(q, k, q_weight, k_weight, positions, cos_sin, q_out, k_out, epsilon=1e-6, interleaved=False):
    """q_out, k_out = rotated norms of q's and k's heads (q_out may be q, k_out may be k)."""
    import torch

    t, d, rot = _check((("q", q, q), ("k", k, k), ("q_out", q_out, q), ("k_out", k_out, k)), q, k,
                       positions, cos_sin, (("q_weight", q_weight, None), ("k_weight", k_weight, None)),
                       epsilon, ("q_out", "k_out"))
    lib = _native.load()
    strides = (ctypes.c_int64 * 8)(q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1),
                                   k.stride(0), k.stride(1), k_out.stride(0), k_out.stride(1))
    with _native.on_device(q.device):
        _native.check(
            lib.bokt_qk_norm_rope(
                q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0, cos_sin.data_ptr(),
                cos_sin.shape[0], q_out.data_ptr(), k_out.data_ptr(), t, q.shape[1], k.shape[1], d,
                rot, strides, 1 if interleaved else 0, float(epsilon), _native.dtype_code(q.dtype),
                _native.current_stream(q.device)),
            "bokt_qk_norm_rope",
        )
    return q_out, k_out


def launch_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, cos_sin, dq, dk, dq_weight,
                    dk_weight, epsilon=1e-6, interleaved=False):
    """Gradients of ``launch``: dq, dk (q's dtype; dq may be dq_out, dk may be
    dk_out) and dq_weight, dk_weight (fp32 [D], overwritten, summed in a fixed
    order: the same inputs give the same bits)."""
    import torch

    t, d, rot = _check(
        (("q", q, q), ("k", k, k), ("dq_out", dq_out, q), ("dk_out", dk_out, k), ("dq", dq, q), ("dk", dk, k)),
        q, k, positions, cos_sin,
        (("q_weight", q_weight, None), ("k_weight", k_weight, None), ("dq_weight", dq_weight, torch.float32),
         ("dk_weight", dk_weight, torch.float32)), epsilon, ("dq", "dk"))
    lib = _native.load()
    strides = (ctypes.c_int64 * 12)()
    for i, (x, dx, g) in enumerate(((q, dq, dq_out), (k, dk, dk_out))):
        strides[6 * i:6 * i + 6] = [x.stride(0), x.stride(1), dx.stride(0), dx.stride(1), g.stride(0),
                                    g.stride(1)]
    with _native.on_device(q.device):
        nbytes = int(lib.bokt_qk_norm_rope_workspace_bytes(d))
        if nbytes < 0:
            _native.check(_native.BOKT_ERR_CUDA_RC, "bokt_qk_norm_rope_workspace_bytes")
        # Fresh per call: calls on other streams and other captured graphs have their own.
        workspace = torch.empty(nbytes // 4, device=q.device, dtype=torch.float32)
        _native.check(
            lib.bokt_qk_norm_rope_backward(
                dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(),
                q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(),
                1 if positions.dtype == torch.int64 else 0, cos_sin.data_ptr(), cos_sin.shape[0],
                dq.data_ptr(), dk.data_ptr(), dq_weight.data_ptr(), dk_weight.data_ptr(), t,
                q.shape[1], k.shape[1], d, rot, strides, 1 if interleaved else 0, float(epsilon),
                _native.dtype_code(q.dtype), workspace.data_ptr(), nbytes,
                _native.current_stream(q.device)),
            "bokt_qk_norm_rope_backward",
        )
    return dq, dk, dq_weight, dk_weight
