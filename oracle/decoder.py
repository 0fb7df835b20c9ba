"""fp64 forms of the decoder-layer operators around attention (numpy, CPU only).

The reference has none of them; these are their definitions:

* ``qk_norm_rope`` / ``qk_norm_rope_backward``: per-head RMSNorm and rotary
  rotation, and its gradients;
* ``lora_gemm``: a shared projection with one low-rank adapter per token;
* ``moe_layer``: top-k softmax gate, gated-SiLU experts, gate-weighted sum.

Every input is taken to fp64 as it is; nothing is rounded in between.
"""

import numpy as np


def rope_table(rows, rot, base=10000.0):
    angle = np.arange(rows, dtype=np.float64)[:, None] * base ** (-np.arange(0, rot, 2) / rot)
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1)


def _pairs(rot, interleaved):
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def _turn(y, cos_sin, positions, interleaved, sign):
    rot = cos_sin.shape[1]
    a, b = _pairs(rot, interleaved)
    c = cos_sin[positions][:, None, : rot // 2].astype(np.float64)
    s = sign * cos_sin[positions][:, None, rot // 2:].astype(np.float64)
    out = y.copy()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def qk_norm_rope(x, w, positions, cos_sin, eps, interleaved=False):
    """x [T, H, D] -> rotated norms, fp64."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return _turn(y, cos_sin, positions, interleaved, 1.0)


def qk_norm_rope_backward(g, x, w, positions, cos_sin, eps, interleaved=False):
    """(dx [T, H, D], dw [D]) for the gradient g of qk_norm_rope's result."""
    x, w, g = (v.astype(np.float64) for v in (x, w, g))
    g = _turn(g, cos_sin, positions, interleaved, -1.0)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, gw = x * r, g * w
    return r * (gw - n * (gw * n).mean(-1, keepdims=True)), (g * n).sum((0, 1))


def lora_gemm(x, w, a, b, scales, ids):
    """x [T, K] @ w [K, N] + scales[i] * (x @ a[i].T) @ b[i] for i = ids[t] >= 0
    (a[i] [rank, K], b[i] [rank, N])."""
    x = x.astype(np.float64)
    out = x @ w.astype(np.float64)
    for i in np.unique(ids[ids >= 0]):
        rows = np.nonzero(ids == i)[0]
        out[rows] += float(scales[i]) * (x[rows] @ a[i].astype(np.float64).T) @ b[i].astype(np.float64)
    return out


def moe_gate(logits, topk, renormalize=True):
    """(ids, gates): the top-k of softmax(logits), ties to the lower index."""
    z = logits.astype(np.float64)
    ids = np.argsort(-z, axis=1, kind="stable")[:, :topk]
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    gates = np.take_along_axis(p, ids, 1)
    return ids, gates / gates.sum(1, keepdims=True) if renormalize else gates


def moe_layer(x, logits, w_gate_up, w_down, topk, renormalize=True):
    """sum_j gate_j (silu(x Wg) * (x Wu)) Wd over each token's experts, fp64;
    w_gate_up [E, K, 2 I] (gate columns first), w_down [E, I, K]."""
    x = x.astype(np.float64)
    inner = w_down.shape[1]
    ids, gates = moe_gate(logits, topk, renormalize)
    out = np.zeros((x.shape[0], w_down.shape[2]))
    for e in np.unique(ids):
        rows, slot = np.nonzero(ids == e)
        gu = x[rows] @ w_gate_up[e].astype(np.float64)
        gate = gu[:, :inner]
        h = gate / (1 + np.exp(-gate)) * gu[:, inner:]
        np.add.at(out, rows, gates[rows, slot][:, None] * (h @ w_down[e].astype(np.float64)))
    return out
