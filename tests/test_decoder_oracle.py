"""The fp64 forms of the decoder-layer operators against differences and brute force (CPU)."""

import numpy as np
import pytest

from oracle import decoder


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [4, 6])
def test_qk_norm_rope_gradients_against_differences(rot, interleaved):
    rng = np.random.default_rng(rot)
    t, h, d, eps, step = 3, 2, 6, 1e-3, 1e-6
    x, g, w = rng.normal(size=(t, h, d)), rng.normal(size=(t, h, d)), rng.normal(size=d)
    table = decoder.rope_table(9, rot)
    pos = np.array([0, 8, 3])

    def loss(x, w):
        return (decoder.qk_norm_rope(x, w, pos, table, eps, interleaved) * g).sum()

    dx, dw = decoder.qk_norm_rope_backward(g, x, w, pos, table, eps, interleaved)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        assert abs((loss(up, w) - loss(down, w)) / (2 * step) - dx[i]) < 1e-7
    for i in range(d):
        up, down = w.copy(), w.copy()
        up[i] += step
        down[i] -= step
        assert abs((loss(x, up) - loss(x, down)) / (2 * step) - dw[i]) < 1e-7


def test_rotation_keeps_lengths_and_depends_on_distance_only():
    rng = np.random.default_rng(1)
    d = 8
    table = decoder.rope_table(100, d)
    w = np.ones(d)
    q, k = rng.normal(size=(1, 1, d)), rng.normal(size=(1, 1, d))
    score = [float((decoder.qk_norm_rope(q, w, np.array([p + 7]), table, 0.0)
                    * decoder.qk_norm_rope(k, w, np.array([p]), table, 0.0)).sum()) for p in (0, 31, 90)]
    assert np.ptp(score) < 1e-12
    assert abs((decoder.qk_norm_rope(q, w, np.array([77]), table, 0.0) ** 2).sum() - d) < 1e-12


def test_moe_gate_ties_and_masked_experts():
    z = np.array([[1.0, 2.0, 2.0, -np.inf], [-np.inf, 0.0, -np.inf, -np.inf]])
    ids, gates = decoder.moe_gate(z, 2)
    assert ids.tolist() == [[1, 2], [1, 0]]
    np.testing.assert_allclose(gates, [[0.5, 0.5], [1.0, 0.0]])


def test_moe_layer_and_lora_by_the_token():
    rng = np.random.default_rng(3)
    t, e, k, inner, top = 5, 4, 6, 3, 2
    x, z = rng.normal(size=(t, k)), rng.normal(size=(t, e))
    gu, dn = rng.normal(size=(e, k, 2 * inner)), rng.normal(size=(e, inner, k))
    out = decoder.moe_layer(x, z, gu, dn, top)
    ids, gates = decoder.moe_gate(z, top)
    for i in range(t):
        want = 0
        for j in range(top):
            y = x[i] @ gu[ids[i, j]]
            want = want + gates[i, j] * ((y[:inner] / (1 + np.exp(-y[:inner])) * y[inner:]) @ dn[ids[i, j]])
        np.testing.assert_allclose(out[i], want, rtol=1e-12)
    a, b, s = rng.normal(size=(3, 2, k)), rng.normal(size=(3, 2, 7)), np.array([0.5, 2.0, 1.0])
    w, who = rng.normal(size=(k, 7)), np.array([2, -1, 0, 2, 1])
    out = decoder.lora_gemm(x, w, a, b, s, who)
    for i, j in enumerate(who):
        want = x[i] @ w + (0 if j < 0 else s[j] * (a[j] @ x[i]) @ b[j])
        np.testing.assert_allclose(out[i], want, rtol=1e-12)
