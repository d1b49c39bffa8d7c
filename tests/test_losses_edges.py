"""Losses over vocabulary logits at the edges of their inputs, against the float64 oracle (oracle/losses.py): values that
are not finite, masses far below a row's largest, labels outside the vocabulary, ids given twice.  The register kernels
and the streaming kernel are reached by the number of rows (streamed: two rows an SM, more than 32 KiB each)."""

import numpy as np
import pytest
import torch

from oracle import losses as oracle

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def _logits(n, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(n, V, generator=g, device="cuda")).to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _cuda(*arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def _device_error():
    import ctypes

    from kdn_b200 import _lib

    code = ctypes.c_int(0)
    assert _lib.load().kdn_device_error(_lib.stream_handle(torch.device("cuda:0")), ctypes.byref(code)) == 0
    return code.value


# ------------------------------------------------------------------------------------------------- NaN in an input
def test_oracle_passes_a_nan_on():
    z, y = np.zeros((3, 4)), np.array([0, 1, -100])
    for bad in ("old", "adv"):
        f = dict(old=np.full(3, -1.0), adv=np.ones(3))
        f[bad][:] = np.nan
        loss, logps, H, d = oracle.policy_loss(z, y, f["old"], f["adv"])
        assert np.isnan(loss) and np.isnan(d[:2]).all() and (d[2] == 0).all()


@gpu
@pytest.mark.parametrize("n,V", [(6, 300), (300, 700), (2, 131072), (300, 16411), (300, 80003)])
@pytest.mark.parametrize("name", ["old_logps", "advantages", "ref_logps"])
@pytest.mark.parametrize("entropy", [0.0, 0.01])
def test_a_nan_in_a_policy_input_reaches_loss_and_gradient(n, V, name, entropy):
    """In a row that counts; in rows that do not (ignored, of weight zero) it changes nothing."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + V)
    z = _logits(n, V, torch.bfloat16, seed=V)
    y = rng.integers(0, V, n)
    w = (0.5 + rng.random(n).astype(np.float32)) / n
    dead = 1 % n
    if n > 2:
        y[2], w[dead] = -100, 0.0
    yd, wd = _cuda(y, w)
    logp = kdn.token_logprobs(z, yd)
    given = dict(old_logps=logp - 0.1, advantages=torch.full_like(logp, 1.5), ref_logps=logp + 0.1)
    call = lambda f, **kw: f(z, yd, given["old_logps"], given["advantages"], ref_logps=given["ref_logps"], kl_coef=0.1,
                             entropy_coef=entropy, **kw)
    clean = call(kdn.policy_loss_and_grad, weights=wd)
    if n > 2:
        given[name][[dead, 2]] = float("nan")
        again = call(kdn.policy_loss_and_grad, weights=wd)
        assert torch.equal(again[0], clean[0]) and torch.equal(again[3], clean[3])
    at = n - 1
    given[name][at] = float("nan")
    for weights in (wd, None):
        loss, logps, H, d = call(kdn.policy_loss_and_grad, weights=weights)
        assert torch.isnan(loss)
        assert torch.isnan(d[at]).all()
        assert torch.equal(logps, clean[1]) and torch.equal(H, clean[2])
        if weights is not None:
            assert torch.equal(d[:at], clean[3][:at])
        assert torch.isnan(call(kdn.policy_loss, weights=weights)[0])
        want = oracle.policy_loss(_np(z[at:]), y[at:], _np(given["old_logps"][at:]), _np(given["advantages"][at:]),
                                  _np(given["ref_logps"][at:]), kl_coef=0.1, entropy_coef=entropy)
        assert np.isnan(want[0]) and np.isnan(want[3]).all()


@gpu
def test_a_ratio_that_overflows_times_no_advantage_is_nothing():
    import kdn_b200 as kdn

    z, y = _logits(4, 300, torch.float32), np.array([3, 5, 7, 9])
    yd, = _cuda(y)
    adv = np.array([0.0, 1.0, 0.0, -0.0], np.float32)
    old = _np(kdn.token_logprobs(z, yd)).astype(np.float32) - np.array([200, 200, 0, 100], np.float32)
    o, a = _cuda(old, adv)
    loss, _, _, d = kdn.policy_loss_and_grad(z, yd, o, a)
    want = oracle.policy_loss(_np(z), y, old, adv)
    assert abs(want[0] + 1.2 / 4) < 1e-6 and abs(float(loss) - want[0]) < 1e-6  # the one clipped ratio, 1 + 0.2
    assert not want[3].any() and not d.any()
