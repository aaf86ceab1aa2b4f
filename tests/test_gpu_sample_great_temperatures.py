"""Sampling at temperatures up to infinity, where every finite logit weighs the
same and a masked one nothing: tokens equal to the 64-bit form's, probabilities
to the bound of test_gpu_sample.py (2^-22 relative, 2^-43 absolute)."""
import numpy as np
import pytest

from test_gpu_sample import check, logits, ops, torch, uniforms  # noqa: F401

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("temperature", [1e30, 1.1e37, 2e37, 1e38, 3.4e38, INF])
@pytest.mark.parametrize("rows,vocab", [(7, 5), (7, 40), (7, 2000), (7, 25000), (90, 1999), (3, 60001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_logits_have_no_weight(device, torch, ops, temperature, rows, vocab, dtype):  # noqa: F811
    x = logits(torch, rows, vocab, vocab, device, "f32", hot=0)
    x[:, 1::2] = -INF
    x[0, 0::4] = float("nan")
    x[1, 2:] = -INF
    x[2] = -INF
    x = x.to(torch.float32 if dtype == "f32" else torch.bfloat16)
    p = np.resize(np.array([0.9, 0.5, 0.05, 0.999, 0.7], np.float32), rows)
    for kw in (dict(top_p=p), dict(top_p=p, min_p=0.3), dict(), dict(top_k=9, top_p=0.6),
               dict(top_k=3000, top_p=0.6), dict(min_p=0.3)):
        tok = check(torch, ops, x, uniforms(rows, vocab), temperature=temperature, **kw)
        assert tok[2] == -1
        live = torch.isfinite(x)[np.arange(rows), np.maximum(tok, 0)].cpu().numpy()
        assert live[np.arange(rows) != 2].all()


@pytest.mark.parametrize("temperature", [3e37, 1e38, 3.4e38])
@pytest.mark.parametrize("rows,vocab", [(4, 2), (4, 1500), (4, 30000), (90, 1999)])
def test_logits_of_the_largest_magnitudes(device, torch, ops, temperature, rows, vocab):  # noqa: F811
    """Finite logits whose differences are beyond f32's largest: their weights
    are exp of a few at such temperatures. (The largest ones stand at both
    ends: 6.8e38 / 3.4e38 = 2.)"""
    x = logits(torch, rows, vocab, vocab, device, "f32", 1.0, hot=0).clamp(-3, 3) * 1e38
    x[:, 0] = torch.finfo(torch.float32).min
    x[:, -1] = torch.finfo(torch.float32).max
    u = uniforms(rows, vocab)
    u[0] = 0.0  # the first logit, the least of all, where nothing cuts it
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.999, min_p=0.001), dict(top_k=9, top_p=0.6),
               dict(top_k=3000, top_p=0.9)):
        tok = check(torch, ops, x, u, temperature=temperature, **kw)
        if not kw and temperature > 5e37:
            assert tok[0] == 0
