"""NativeKhqLayer.attention_prefill, the many-token form of attention_step: its
front against the steps' own, its attention against prefill on that front."""
import numpy as np
import pytest
import torch

from khq import dump, paged
from khq.centroids import synthetic_layer
from khq.layer import ROPE_BASE, KhqOptions, NativeKhqLayer

pytestmark = pytest.mark.gpu

H_Q, H_KV, D = 24, 4, 256
SCALE, EPS = 1.0 / 16.0, 1e-6


def layer(cap=1024):
    return NativeKhqLayer(synthetic_layer(3, seed=1234), H_q=H_Q, H_kv=H_KV, cap=cap,
                          options=KhqOptions(splits=16, fused=True))


def ring(lay, which, slot):
    from test_gpu_layer import _hip_d2d

    t = torch.empty((H_KV, D), device="cuda", dtype=torch.float16)
    assert _hip_d2d(t.data_ptr(), lay.payload_ptrs()[which] + slot * t.numel() * 2, t.numel() * 2) == 0
    return t


def inputs(n, weights, device, seed=0):
    rng = np.random.default_rng(seed)
    t = [torch.from_numpy((rng.standard_normal(s) * 3).astype(np.float16)).to(device)
         for s in ((n, H_Q, 2 * D), (n, H_KV, D), (n, H_KV, D))]
    w = [torch.from_numpy(rng.uniform(0.5, 1.5, D).astype(np.float32)).to(device) if weights else None
         for _ in range(2)]
    return t, w


def close(got, want, pos):
    """Rotated heads [n][heads][D] whose normalised values may each be the next one of the
    type (a step is 2^-10 of a value at most) and which are rounded once more on either side
    (half a step each): a pair of size r turns them into r (sqrt(2) + 1) 2^-10.  The steps'
    angles are of 32 bits: the exponent, at most 16.1, is off by a step of 2^-19 of the
    logarithm, half of one of the product and 16.1 x 2^-24 of its fraction, the exponential
    by 2 x 2^-23 and the angle by 2^-24 relative: less than 4.2e-6 pos r, frequencies being 1
    or less.  Dims past the 64th: a step.  (Values below 2^-14 have steps of 2^-24.)"""
    got, want = got.double(), want.double()
    x0, x1 = want[..., :32], want[..., 32:64]
    r = torch.sqrt(x0 * x0 + x1 * x1)
    tol = r * (2.4143 * 2.0 ** -10 + 4.2e-6 * pos[:, None, None]) + 2.0 ** -22
    assert bool(((got[..., :32] - x0).abs() <= tol).all())
    assert bool(((got[..., 32:64] - x1).abs() <= tol).all())
    rest = want[..., 64:]
    assert bool(((got[..., 64:] - rest).abs() <= rest.abs() * 2.0 ** -10 + 2.0 ** -23).all())


@pytest.mark.parametrize("n,pos0,weights", [(1, 0, False), (1, 37, True), (300, 0, True), (129, 250, False)])
def test_front_is_the_steps(device, n, pos0, weights):
    (q_gate, k, v), (qw, kw) = inputs(n, weights, device, n)
    A, B = layer(), layer()
    q1, k1 = q_gate.clone(), k.clone()
    out = torch.empty((n, H_Q, D), device=device, dtype=torch.float16)
    for i in range(n):
        assert A.attention_step(q1[i], k1[i], v[i], out[i], SCALE, pos=pos0 + i, q_norm_w=qw,
                                k_norm_w=kw, eps=EPS)
    q2, k2, v2 = q_gate.clone(), k.clone(), v.clone()
    out2 = torch.empty_like(out)
    assert B.attention_prefill(q2, k2, v2, out2, SCALE, pos=pos0, q_norm_w=qw, k_norm_w=kw,
                               eps=EPS) == n
    pos = pos0 + torch.arange(n, device=device, dtype=torch.float64)
    close(q2[..., :D], q1[..., :D], pos)
    close(k2, k1, pos)
    assert torch.equal(q2[..., D:], q_gate[..., D:]) and torch.equal(v2, v)
    assert A.state()[:2] == B.state()[:2]
    for i in range(max(0, n - 256), n, 13):
        u, w = ring(B, 10, i % 256).double(), ring(A, 10, i % 256).double()
        assert bool(((u - w).abs() <= w.abs() * 2.0 ** -10 + 2.0 ** -23).all())  # a step
        assert torch.equal(ring(B, 8, i % 256), k2[i]) and torch.equal(ring(B, 9, i % 256), v[i])


@pytest.mark.parametrize("n", [1, 300])
def test_attention_is_that_of_prefill(device, n):
    (q_gate, k, v), (qw, kw) = inputs(n, True, device, 5)
    A, B = layer(), layer()
    outs = [torch.empty((n, H_Q, D), device=device, dtype=torch.float16) for _ in range(2)]
    q1, k1, u = q_gate.clone(), k.clone(), torch.empty_like(k)
    paged.qk_norm_rope(q1[..., :D], k1, q1[..., :D], pos0=11, q_weight=qw, k_weight=kw, eps=EPS,
                       theta=ROPE_BASE, k_out=k1, k_normed=u, round_norm=True)
    A.prefill(q1, k1, v, u, outs[0], SCALE)
    B.attention_prefill(q_gate, k, v, outs[1], SCALE, pos=11, q_norm_w=qw, k_norm_w=kw, eps=EPS)
    assert torch.equal(outs[0], outs[1])
    # and what it leaves behind: the next token's step
    (q, kk, vv), _ = inputs(1, False, device, 6)
    last = [torch.empty((H_Q, D), device=device, dtype=torch.float16) for _ in range(2)]
    for lay, o in zip((A, B), last):
        lay.attention_step(q[0].clone(), kk[0].clone(), vv[0], o, SCALE, pos=11 + n, eps=EPS)
    assert torch.equal(*last)


def test_refusals(device, tmp_path):
    (q, k, v), _ = inputs(2, False, device)
    out = torch.empty((2, H_Q, D), device=device, dtype=torch.float16)
    lay = layer()
    for bad in (dict(q_gate=q.float()), dict(k=k.cpu()), dict(v=v[:1]), dict(out=out[:, ::2])):
        a = dict(q_gate=q, k=k, v=v, out=out) | bad
        with pytest.raises((TypeError, ValueError)):
            lay.attention_prefill(*a.values(), SCALE, pos=0)
    with pytest.raises(ValueError):
        lay.attention_prefill(q, k, v, out, SCALE, pos=0, q_norm_w=torch.ones(64, device=device))
    lay.set_dump(dump.Recorder(str(tmp_path), max_tokens=64, kv_dim=H_KV * D), layer_id=3)
    with pytest.raises(RuntimeError):
        lay.attention_prefill(q, k, v, out, SCALE, pos=0)
    lay.set_dump(None, 0)
    assert lay.state()[:2] == (0, 0)
