"""RMS norm of q and k heads with rotation against the formula in fp64.

Tolerance: the mean of D squares (D / 2 steps of 2^-24 relative, halved by the
square root), rsqrt (2 units), four products and one sum per element: below
(D / 4 + 8) * 2^-24 of |y cos| + |y' sin|, plus half a unit of the output type.
"""

import numpy as np
import pytest
import torch

import infrared_b200 as irb
from oracle import kv_q8_np as q8

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda"


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().double().cpu().numpy()


def tables(rng, n, d):
    ang = rng.uniform(0, 30000, size=(n, 1)) * 1e6 ** (-np.arange(0, d, 2) / d)
    ang = np.concatenate([ang, ang], axis=1)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def check(got, x, w, cos, sin, eps):
    x, wh = host(x), None if w is None else host(w)
    want = q8.norm_rope(x, wh, cos, sin, eps)
    size = q8.norm_rope(np.abs(x), None if wh is None else np.abs(wh), np.abs(cos), np.abs(sin), eps)
    y = np.abs(x) / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * (1 if wh is None else np.abs(wh))
    half = x.shape[-1] // 2
    other = np.concatenate([y[..., half:], y[..., :half]], -1)
    size = y * np.abs(cos)[:, None] + other * np.abs(sin)[:, None]
    fi = torch.finfo(got.dtype)
    tol = (x.shape[-1] / 4 + 8) * 2.0 ** -24 * size + fi.eps / 2 * np.abs(want) * (1 + 2.0 ** -6) + \
        fi.tiny * fi.eps
    assert (np.abs(host(got) - want) <= tol).all(), float((np.abs(host(got) - want) - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,h,hkv,d", [
    (1, 1, 1, 64), (1, 28, 4, 128), (3, 14, 2, 64), (64, 28, 4, 128), (257, 7, 1, 128),
    (1000, 5, 3, 64), (33, 64, 64, 128),
])
def test_norm_rope(n, h, hkv, d, dtype):
    rng = np.random.default_rng(n + h)
    qkv = dev(rng.normal(size=(n, (h + 2 * hkv) * d)) * 3).to(dtype)
    q, k = qkv[:, :h * d].view(n, h, d), qkv[:, h * d:(h + hkv) * d].view(n, hkv, d)
    q[0, 0] = 0.0
    wq, wk = dev(1 + rng.normal(size=d)).to(dtype), dev(rng.normal(size=d)).to(dtype)
    cos, sin = tables(rng, n, d)
    before = qkv.clone()
    for a, b in ((wq, wk), (None, wk), (None, None)):
        qo, ko = irb.qk_norm_rope(q, k, a, b, dev(cos), dev(sin), 1e-6)
        check(qo, q, a, cos, sin, 1e-6)
        check(ko, k, b, cos, sin, 1e-6)
    assert torch.equal(qkv, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_place_and_strided(dtype):
    rng = np.random.default_rng(0)
    n, h, hkv, d = 21, 6, 2, 64
    for pad in (0, 3, 8):   # 3: rows that no vector load can take
        row = (h + 2 * hkv) * d + pad
        x = dev(rng.normal(size=(n, row))).to(dtype)
        q, k = x[:, :h * d].view(n, h, d), x[:, h * d:(h + hkv) * d].view(n, hkv, d)
        w = dev(rng.normal(size=d + 1)).to(dtype)[1:] if pad == 3 else dev(rng.normal(size=d)).to(dtype)
        cs = dev(rng.normal(size=(n, 2 * d)).astype(np.float32))
        cos, sin = cs[:, :d], cs[:, d:]
        qo, ko = irb.qk_norm_rope(q, k, w, w, cos, sin, 1e-5)
        check(qo, q, w, host(cos).astype(np.float32), host(sin).astype(np.float32), 1e-5)
        y = x.clone()
        q2, k2 = y[:, :h * d].view(n, h, d), y[:, h * d:(h + hkv) * d].view(n, hkv, d)
        r = irb.qk_norm_rope(q2, k2, w, w, cos, sin, 1e-5, q_out=q2, k_out=k2)
        assert r[0] is q2 and torch.equal(q2, qo) and torch.equal(k2, ko)
        assert torch.equal(y[:, (h + hkv) * d:], x[:, (h + hkv) * d:])   # V stays


def test_empty_graph_and_refusals():
    q = torch.randn(4, 3, 64, device=DEV)
    k = torch.randn(4, 1, 64, device=DEV)
    cos, sin = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV)
    a, b = irb.qk_norm_rope(q[:0], k[:0], None, None, cos[:0], sin[:0], 1e-6)
    assert a.shape == (0, 3, 64) and b.shape == (0, 1, 64)
    want = irb.qk_norm_rope(q, k, None, None, cos, sin, 1e-6)
    g = torch.cuda.CUDAGraph()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    with torch.cuda.graph(g):
        irb.qk_norm_rope(q, k, None, None, cos, sin, 1e-6, q_out=qo, k_out=ko)
    g.replay()
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    for bad in (lambda: irb.qk_norm_rope(q, k.half(), None, None, cos, sin, 1e-6),
                lambda: irb.qk_norm_rope(q, k[:3], None, None, cos, sin, 1e-6),
                lambda: irb.qk_norm_rope(q, k, torch.ones(32, device=DEV), None, cos, sin, 1e-6),
                lambda: irb.qk_norm_rope(q, k, None, None, cos.half(), sin, 1e-6),
                lambda: irb.qk_norm_rope(q, k, None, None, cos[:, :32], sin[:, :32], 1e-6),
                lambda: irb.qk_norm_rope(q.transpose(1, 2), k, None, None, cos, sin, 1e-6)):
        with pytest.raises(ValueError):
            bad()
