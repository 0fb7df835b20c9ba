"""A whole mixture-of-experts layer for a few tokens, in two kernels (sm_100a).

For the decode batches of a served model: where the routed chain
(``moe_routing.topk_gate``, ``MoeRouter``, ``gather_rows``,
``moe_grouped_gemm.launch`` twice, the activation, ``combine``) is bound by its
launches, ``launch`` runs the layer from router logits to combined output at
the rate at which the weights of the experts in use arrive from HBM:

    p = softmax(logits[t]);  e_1..e_k the k largest (ties to the lower index)
    out[t] = sum_j g_j (silu(x[t] @ Wg[e_j]) * (x[t] @ Wu[e_j])) @ Wd[e_j]

with ``w_gate_up`` [E, K, 2 I] holding the gate columns and then the up columns
of every expert, ``w_down`` [E, I, K], and g_j = p[e_j], divided by their sum
with ``renormalize``.  The reference has the grouped product alone
(``bo_kernel_tuner/kernels/moe_grouped_gemm.py:61-65``) and leaves the rest of
the layer outside.
"""

from flashattentionanycard_b200 import _native

MAX_TOKENS, MAX_TOPK, MAX_EXPERTS = 128, 8, 1024


def workspace_bytes(tokens, experts, k, inner, topk):
    """Device scratch of one call on the current device (contents free before and after)."""
    lib = _native.load()
    n = int(lib.bokt_moe_decode_workspace_bytes(int(tokens), int(experts), int(k), int(inner), int(topk)))
    if n < 0:
        raise RuntimeError(f"bokt_moe_decode_workspace_bytes: {lib.bokt_last_error().decode()}")
    return n


def launch(x, logits, w_gate_up, w_down, out, topk, renormalize=True, workspace=None):
    """out[T, K] = the layer's output for x [T, K] and logits [T, E] (T <= 128).

    ``workspace``: a uint8 tensor of ``workspace_bytes`` (calls that may overlap
    on the GPU need one each); by default the call takes a fresh one from
    torch's allocator."""
    import torch

    if x.dim() != 2 or w_gate_up.dim() != 3 or w_down.dim() != 3 or logits.dim() != 2:
        raise ValueError("x and logits must have two dimensions, the weights three")
    t, k = x.shape
    e, inner = w_gate_up.shape[0], w_down.shape[1]
    topk = int(topk)
    if w_gate_up.shape != (e, k, 2 * inner) or w_down.shape != (e, inner, k):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w_gate_up {tuple(w_gate_up.shape)} "
                         f"(expected [E, K, 2 I]), w_down {tuple(w_down.shape)} (expected [E, I, K])")
    if logits.shape != (t, e) or out.shape != (t, k):
        raise ValueError(f"shape mismatch: logits {tuple(logits.shape)}, out {tuple(out.shape)}")
    if not 1 <= topk <= min(e, MAX_TOPK):
        raise ValueError(f"topk must be in [1, {min(e, MAX_TOPK)}], got {topk}")
    if t > MAX_TOKENS or e > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_TOKENS} tokens and {MAX_EXPERTS} experts (got {t} and {e}): "
                         "larger batches go through moe_routing and moe_grouped_gemm")
    if k % 8 or inner % 8:
        raise ValueError(f"K and I must be multiples of 8 (got {k} and {inner})")
    if not (x.dtype == w_gate_up.dtype == w_down.dtype == out.dtype):
        raise ValueError("x, the weights and out must share one dtype")
    if logits.dtype == torch.float32:
        logits_dtype = 2
    else:
        logits_dtype = _native.dtype_code(logits.dtype)
    dtype = _native.dtype_code(x.dtype)
    tensors = (x, logits, w_gate_up, w_down, out)
    if not all(v.is_contiguous() for v in tensors):
        raise ValueError("x, logits, the weights and out must be contiguous")
    device = x.device
    if not (x.is_cuda and all(v.device == device for v in tensors)):
        raise ValueError("all tensors must be on one CUDA device")
    lib = _native.load()
    with _native.on_device(device):
        need = lib.bokt_moe_decode_workspace_bytes(t, e, k, inner, topk)
        if need < 0:
            raise RuntimeError(f"bokt_moe_decode: {lib.bokt_last_error().decode()}")
        if workspace is None:
            workspace = torch.empty(need, device=device, dtype=torch.uint8)
        elif workspace.device != device or not workspace.is_contiguous() \
                or workspace.numel() * workspace.element_size() < need:
            raise ValueError(f"workspace must be a contiguous tensor of {need} bytes on {device}")
        _native.check(
            lib.bokt_moe_decode(
                x.data_ptr(), logits.data_ptr(), logits_dtype, w_gate_up.data_ptr(), w_down.data_ptr(),
                out.data_ptr(), t, e, k, inner, topk, 1 if renormalize else 0, dtype,
                workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                _native.current_stream(device)),
            "bokt_moe_decode",
        )
    return out
