"""Losses over vocabulary logits (kdn_b200.kernels.losses) against the float64 oracle (oracle/losses.py).

CPU: the oracle's gradients against central differences, argument checks of the C entries, refusals of the Python
surface.  GPU: every operator over sizes, types, row layouts and masks.

Tolerances.  With X = max |z - row max| / T, the fp32 exponent (z - m) log2(e) / T carries a relative error of
2^-23 (the rounded factor and one multiply-add), the base-2 exponential 2^-22 and the sum of V terms, in a tree over
at most 64 values a lane, 2^-18: a log-probability is within eps = 2^-23 X + 2^-17 of its value, and a probability
within that share of its own.  A gradient element c (1[y] - q) / T adds the error of c, itself a function of the
log-probability with slope at most |c| (1 + |advantage|): 8 eps of the row's largest coefficient bounds it; bf16
gradients add half a unit of the last place, at most 2^-8 of the value.
"""

import numpy as np
import pytest
import torch

from oracle import losses as oracle

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
LAYOUTS = ["packed", "padded", "offset", "strided"]


# ----------------------------------------------------------------------------------------------------- the oracle
def _differences(f, z, d, step=1e-5):
    return (f(z + step * d) - f(z - step * d)) / (2 * step)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
def test_oracle_gradients_are_differences(temperature):
    rng = np.random.default_rng(0)
    n, V, K = 6, 23, 5
    z = 2 * rng.standard_normal((n, V))
    y = rng.integers(0, V, n)
    y[2] = -100
    up = rng.standard_normal(n)
    old, adv, ref, w = (rng.standard_normal(n) - s for s in (3.0, 0.0, 3.0, -2.0))
    t, ids = rng.standard_normal((n, K)), np.stack([rng.permutation(V)[:K] for _ in range(n)])
    ids[4, 0] = -1
    lse = np.log(np.exp(t / temperature).sum(-1)) + 0.2
    cu = [0, 2, 2, 5, 6]
    losses = [
        (lambda x: (oracle.token_logprobs(x, y, up, temperature)[0] * up).sum(),
         oracle.token_logprobs(z, y, up, temperature)[-1]),
        (lambda x: oracle.policy_loss(x, y, old, adv, ref, w, 0.2, 0.3, 0.1, 0.05, temperature)[0],
         oracle.policy_loss(z, y, old, adv, ref, w, 0.2, 0.3, 0.1, 0.05, temperature)[-1]),
        (lambda x: oracle.preference_loss(x, y, cu, ref, 0.5, 0.1, False, temperature)[0],
         oracle.preference_loss(z, y, cu, ref, 0.5, 0.1, False, temperature)[-1]),
        (lambda x: oracle.preference_loss(x, y, cu, None, 0.5, 0.0, True, temperature)[0],
         oracle.preference_loss(z, y, cu, None, 0.5, 0.0, True, temperature)[-1]),
        (lambda x: oracle.distillation_loss(x, t, ids, None, w, temperature)[0],
         oracle.distillation_loss(z, t, ids, None, w, temperature)[-1]),
        (lambda x: oracle.distillation_loss(x, t, ids, lse, None, temperature)[0],
         oracle.distillation_loss(z, t, ids, lse, None, temperature)[-1]),
    ]
    for f, g in losses:
        for _ in range(3):
            d = rng.standard_normal((n, V))
            # central differences at step 1e-5: error ~1e-10 (third derivative) + 1e-16 / 1e-5
            assert abs(_differences(f, z, d) - (g * d).sum()) < 1e-7


# ------------------------------------------------------------------------------------------------------- refusals
def test_loss_argument_checks(lib):
    P, Q, S = 4096, 1 << 30, 1 << 24
    big = 1 << 30
    lp = lambda **kw: lib.kdn_token_logprobs(*[kw.get(k, d) for k, d in (
        ("z", P), ("dt", 1), ("ld", 100), ("y", P), ("it", 1), ("ig", -100), ("lp", P), ("st", None), ("n", 4),
        ("V", 100), ("T", 1.0))], None)
    assert lp(n=0) == 0                       # nothing to do
    assert lp(dt=2) == 1 and lp(it=3) == 1    # bad types
    assert lp(ld=99) == 1                     # rows overlap
    assert lp(V=0) == 1 and lp(n=-1) == 1
    assert lp(z=None) == 1 and lp(y=None) == 1 and lp(lp=None) == 1
    assert lp(z=P + 1) == 1                   # not aligned to an element
    assert lp(T=0.0) == 1 and lp(T=-1.0) == 1 and lp(T=float("nan")) == 1 and lp(T=float("inf")) == 1
    bw = lambda **kw: lib.kdn_token_logprobs_backward(*[kw.get(k, d) for k, d in (
        ("z", P), ("dt", 1), ("ld", 100), ("y", P), ("it", 1), ("ig", -100), ("st", P), ("d", P), ("g", Q),
        ("ldd", 100), ("n", 4), ("V", 100), ("T", 1.0))], None)
    assert bw(n=0) == 0
    assert bw(st=None) == 1 and bw(d=None) == 1 and bw(g=None) == 1
    assert bw(ldd=99) == 1 and bw(g=Q + 1) == 1
    assert bw(g=P + 4) == 1                   # the gradient overlaps the logits
    assert b"overlap" in lib.kdn_last_error()
    po = lambda **kw: lib.kdn_policy_loss(*[kw.get(k, d) for k, d in (
        ("z", P), ("dt", 1), ("ld", 100), ("y", P), ("it", 1), ("ig", -100), ("old", P), ("adv", P), ("ref", None),
        ("w", None), ("lo", 0.2), ("hi", 0.2), ("kl", 0.0), ("ent", 0.0), ("T", 1.0), ("loss", P), ("lp", P),
        ("H", None), ("g", Q), ("ldd", 100), ("n", 4), ("V", 100), ("ws", 256), ("wsb", big))], None)
    assert po(lo=1.5) == 1 and po(hi=-0.1) == 1 and po(lo=float("nan")) == 1
    assert po(kl=0.1) == 1                    # a KL term without a reference
    assert po(kl=float("nan")) == 1 and po(ent=float("nan")) == 1
    assert po(old=None) == 1 and po(adv=None) == 1 and po(loss=None) == 1
    assert po(wsb=16) == 4 and po(ws=None) == 4 and po(ws=264) == 1
    assert lib.kdn_policy_loss_workspace_size(4) == 512 and lib.kdn_policy_loss_workspace_size(-1) == 0
    assert lib.kdn_distillation_loss_workspace_size(65) == 768
    assert lib.kdn_preference_loss_workspace_size(33, 65) == 256 + 512 + 256 + 512
    pr = lambda **kw: lib.kdn_preference_loss(*[kw.get(k, d) for k, d in (
        ("z", P), ("dt", 1), ("ld", 100), ("y", P), ("it", 1), ("ig", -100), ("cu", P), ("pairs", 2), ("ref", None),
        ("beta", 0.1), ("eps", 0.0), ("norm", 0), ("T", 1.0), ("loss", P), ("lr", P), ("lp", P), ("g", Q),
        ("ldd", 100), ("n", 4), ("V", 100), ("ws", 256), ("wsb", big))], None)
    assert pr(pairs=0) == 1 and pr(beta=0.0) == 1 and pr(eps=0.5) == 1 and pr(eps=-0.1) == 1
    assert pr(cu=None) == 1 and pr(lr=None) == 1 and pr(wsb=16) == 4
    di = lambda **kw: lib.kdn_distillation_loss(*[kw.get(k, d) for k, d in (
        ("z", P), ("dt", 1), ("ld", 100), ("t", P), ("tt", 0), ("ids", P), ("it", 1), ("K", 8), ("lse", None),
        ("w", None), ("T", 1.0), ("loss", P), ("kl", P), ("g", Q), ("ldd", 100), ("n", 4), ("V", 100), ("ws", 256),
        ("wsb", big))], None)
    assert di(K=0) == 1 and di(K=1025) == 2 and di(tt=7) == 1
    assert di(t=None) == 1 and di(ids=None) == 1 and di(kl=None) == 1 and di(wsb=16) == 4
    assert lib.kdn_scale_rows(P, 1, 100, 0, 100, P, None) == 0
    assert lib.kdn_scale_rows(P, 1, 100, 4, 100, None, None) == 1
    assert lib.kdn_scale_rows(P, 1, 50, 4, 100, P, None) == 1


def test_losses_have_no_cpu_path():
    import kdn_b200 as kdn

    z, y = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    f = torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA"):
        kdn.token_logprobs(z, y)
    with pytest.raises(RuntimeError, match="CUDA"):
        kdn.policy_loss(z, y, f, f)
    with pytest.raises(RuntimeError, match="CUDA"):
        kdn.preference_loss(z, y, torch.tensor([0, 1, 2]))
    with pytest.raises(RuntimeError, match="CUDA"):
        kdn.distillation_loss(z, z[:, :2], torch.zeros(2, 2, dtype=torch.int64))


@gpu
def test_losses_refuse_wrong_tensors():
    import kdn_b200 as kdn

    z = torch.zeros(2, 8, device="cuda")
    y = torch.zeros(2, dtype=torch.int64, device="cuda")
    f = torch.zeros(2, device="cuda")
    for bad in (lambda: kdn.token_logprobs(z.half(), y), lambda: kdn.token_logprobs(z[0], y),
                lambda: kdn.token_logprobs(z, y[:1]), lambda: kdn.token_logprobs(z, f),
                lambda: kdn.token_logprobs(z, y.cpu()), lambda: kdn.token_logprobs(z, y, temperature=0.0),
                lambda: kdn.policy_loss(z, y, f, f[:1]), lambda: kdn.policy_loss(z, y, y, f),
                lambda: kdn.policy_loss(z, y, f, f, kl_coef=0.1), lambda: kdn.policy_loss(z, y, None, f),
                lambda: kdn.policy_loss(z, y, f, f, clip_low=2.0),
                lambda: kdn.preference_loss(z, y, torch.tensor([0, 2], device="cuda")),
                lambda: kdn.preference_loss(z, y, torch.tensor([0, 1, 2, 2], device="cuda")),
                lambda: kdn.preference_loss(z, y, torch.tensor([0, 1, 2])),
                lambda: kdn.preference_loss(z[None], y[None], torch.tensor([0, 1, 2], device="cuda")),
                lambda: kdn.distillation_loss(z, z[:, :2], y), lambda: kdn.distillation_loss(z, z[:1, :2], y),
                lambda: kdn.distillation_loss(z, z[:, :0], y.view(2, 1)[:, :0]),
                lambda: kdn.distillation_loss(z, torch.zeros(2, 1025, device="cuda"),
                                              torch.zeros(2, 1025, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------------------------------------------------- inputs
def _logits(n, V, dtype, layout, seed=0, scale=3.0):
    """Logits [n, V] whose rows start on 16 bytes (padded), wherever V leaves them (packed), one element past that
    (offset), or 5 elements further apart than V (strided)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per16 = 16 // torch.empty((), dtype=dtype).element_size()
    ld = {"padded": -(-V // per16) * per16, "strided": V + 5}.get(layout, V)
    flat = (scale * torch.randn(n * ld + 1, generator=g, device="cuda")).to(dtype)
    flat = flat[1:] if layout == "offset" else flat[:-1]
    return flat.view(n, ld)[:, :V]


def _np(t):
    return t.detach().double().cpu().numpy()


def _eps(z, temperature):
    zz = _np(z)
    with np.errstate(invalid="ignore"):
        fin = np.where(np.isfinite(zz), zz, np.nan)
        X = np.nanmax(np.nanmax(fin, -1) - np.nanmin(fin, -1)) / temperature
    return 2.0 ** -23 * X + 2.0 ** -17


def _assert_grad(got, ref, coef, eps, dtype):
    """|got - ref| <= 8 eps max|coef of the row| (+ half a bf16 unit of the value)"""
    got = _np(got)
    tol = 8 * eps * np.abs(coef)[:, None] + (2.0 ** -8 + 1e-6) * np.abs(ref) * (dtype == torch.bfloat16) + 1e-38
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    bad = ~((np.abs(got - ref) <= tol) | np.isnan(ref))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], ref[bad][:4])


def _labels(n, V, rng, index=torch.int64, ignored=0):
    y = rng.integers(0, V, n)
    y[rng.permutation(n)[:ignored]] = -100
    return y, torch.from_numpy(y).to("cuda", index)


SIZES = [(1, 1), (3, 2), (5, 7), (17, 31), (33, 200), (4, 1000), (9, 4099), (300, 4096), (7, 32000), (2, 50021),
         (3, 131072), (1, 262145), (2, 300007)]


# rows enough, and long enough, for the kernel that streams them (two rows an SM, more than 32 KiB each), on one CTA a
# row and on a cluster; every layout of the others
STREAM = [(300, 16411, torch.bfloat16, "packed"), (300, 8200, torch.float32, "offset"),
          (311, 40001, torch.bfloat16, "strided"), (300, 40000, torch.float32, "padded"),
          (297, 80003, torch.bfloat16, "offset"), (297, 80003, torch.float32, "packed")]


# ----------------------------------------------------------------------------------------------- log-probabilities
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,V", SIZES)
def test_token_logprobs(n, V, layout, dtype):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + V)
    T = [1.0, 0.7, 2.0][(n + V) % 3]
    z = _logits(n, V, dtype, layout, seed=V)
    y, yd = _labels(n, V, rng, [torch.int64, torch.int32][V % 2], ignored=n // 3)
    up = rng.standard_normal(n).astype(np.float32)
    ref, dref = oracle.token_logprobs(_np(z), y, up, T)
    eps = _eps(z, T)
    got = kdn.token_logprobs(z, yd, temperature=T)
    assert got.shape == (n,) and got.dtype == torch.float32
    assert np.abs(_np(got) - ref).max() <= eps
    zg = z.detach().requires_grad_()
    logps = kdn.token_logprobs(zg, yd, temperature=T)
    assert torch.equal(logps, got)
    (d,) = torch.autograd.grad(logps, zg, torch.from_numpy(up).cuda())
    assert d.shape == z.shape and d.dtype == dtype
    _assert_grad(d, dref, up / T, eps, dtype)
    (d2,) = torch.autograd.grad(kdn.token_logprobs(zg, yd, temperature=T), zg, torch.from_numpy(up).cuda())
    assert torch.equal(d, d2)


@gpu
def test_token_logprobs_leading_dims_and_streams():
    import kdn_b200 as kdn

    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(2, 5, 333, generator=g, device="cuda")
    y = torch.randint(0, 333, (2, 5), generator=g, device="cuda")
    flat = kdn.token_logprobs(z.view(10, 333), y.view(10))
    assert torch.equal(kdn.token_logprobs(z, y), flat.view(2, 5))
    # rows of another order lie elsewhere within 16 bytes (V is odd): sums in another order, within eps
    other = kdn.token_logprobs(z.transpose(0, 1), y.t())
    assert float((other - flat.view(2, 5).t()).abs().max()) <= 2 * _eps(z.view(10, 333), 1.0)
    assert torch.equal(kdn.token_logprobs(z[0].t().contiguous().t(), y[0]), flat[:5])      # columns not adjacent
    wide = torch.stack([y.view(10), y.view(10)], 1)[:, 0]                                   # strided labels
    assert torch.equal(kdn.token_logprobs(z.view(10, 333), wide), flat)
    same = kdn.token_logprobs(z[:1, :1].expand(1, 4, 333), y[:1, :1].expand(1, 4))          # one row, four times
    assert torch.equal(same, flat[:1].expand(1, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = kdn.token_logprobs(z, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, flat.view(2, 5))
    assert kdn.token_logprobs(z[:0], y[:0]).shape == (0, 5)
    zg = z.clone().requires_grad_()
    (kdn.token_logprobs(zg * 1.0, y) * 2).sum().backward()
    p = torch.softmax(z.double(), -1)
    ref = 2 * (torch.nn.functional.one_hot(y, 333) - p)
    assert float((zg.grad - ref).abs().max()) < 16 * _eps(z.view(10, 333), 1.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 515, 40000])
def test_masked_infinite_and_nan_logits(V, dtype):
    """-inf logits have probability zero; a row of nothing else, with a NaN or with +inf gives NaN; ignored rows give
    zeros whatever they hold; a masked label gives -inf and a finite gradient."""
    import kdn_b200 as kdn

    inf = float("inf")
    z = _logits(8, V, dtype, "packed", seed=1).clone()
    z[0, 1::2] = -inf                       # half of the vocabulary masked
    z[1, :] = -inf                          # nothing left
    z[2, V // 2] = float("nan")
    z[3, V - 1] = inf
    z[4, :] = float("nan")                  # ignored
    z[5, :-1] = -inf                        # one entry left
    z[6, :] = torch.finfo(dtype).min        # the type's lowest value everywhere: a uniform row
    z[7, 3] = -inf                          # the label itself masked
    y = np.array([0, 0, 0, 0, -100, V - 1, 2, 3])
    up = np.array([1.0, 1.0, 1.0, 1.0, 1.0, -2.0, 0.5, 1.0], np.float32)
    zg = z.requires_grad_()
    logps = kdn.token_logprobs(zg, torch.from_numpy(y).cuda())
    (d,) = torch.autograd.grad(logps, zg, torch.from_numpy(up).cuda())
    ref, dref = oracle.token_logprobs(_np(z), y, up)
    got, eps = _np(logps), 2.0 ** -23 * 40 + 2.0 ** -17
    assert np.isnan(got[1:4]).all() and np.isnan(ref[1:4]).all()
    assert got[4] == 0.0 and got[5] == 0.0 and got[7] == -inf
    assert abs(got[0] - ref[0]) <= eps and abs(got[6] + np.log(V)) <= eps
    assert not np.isnan(_np(d)[4]).any() and (_np(d)[4] == 0).all()
    assert np.isnan(_np(d)[1:4]).all()
    rows = [0, 5, 6, 7]
    _assert_grad(d[rows], dref[rows], up[rows], eps, dtype)
    # logits far from zero lose nothing: the statistics are relative to the row's maximum
    far = (_logits(4, V, torch.float32, "packed", seed=2).round() + 2.0 ** 14)
    yd = torch.zeros(4, dtype=torch.int64, device="cuda")
    assert torch.equal(kdn.token_logprobs(far, yd), kdn.token_logprobs(far - 2.0 ** 14, yd))


@gpu
def test_labels_outside_the_vocabulary_are_recorded():
    import ctypes

    import kdn_b200 as kdn
    from kdn_b200 import _lib

    code = ctypes.c_int(0)
    read = lambda: (_lib.load().kdn_device_error(_lib.stream_handle(torch.device("cuda:0")), ctypes.byref(code)),
                    code.value)
    assert read()[0] == 0
    z = _logits(3, 100, torch.float32, "packed").requires_grad_()
    logps = kdn.token_logprobs(z, torch.tensor([100, 5, -7], device="cuda"))
    (d,) = torch.autograd.grad(logps.sum(), z)
    assert logps[0] == 0 and logps[2] == 0 and logps[1] != 0
    assert (d[0] == 0).all() and (d[2] == 0).all() and (d[1] != 0).any()
    assert read() == (0, 1) and read() == (0, 0)
    t, ids = torch.randn(1, 4, device="cuda"), torch.tensor([[3, 100, 7, 5]], device="cuda")
    kl = kdn.distillation_loss(z[:1].detach(), t, ids)[1]
    ids[0, 1] = -1  # an id outside the vocabulary is skipped, as padding is
    assert torch.equal(kl, kdn.distillation_loss(z[:1].detach(), t, ids)[1])
    assert read() == (0, 1)
    kdn.preference_loss(z.detach(), torch.zeros(3, dtype=torch.int64, device="cuda"),
                        torch.tensor([0, 2, 9], device="cuda"))
    assert read() == (0, 1) and read() == (0, 0)


# ----------------------------------------------------------------------------------------------------- policy loss
def _policy_inputs(n, V, dtype, layout, rng, seed, ignored):
    z = _logits(n, V, dtype, layout, seed=seed)
    y, yd = _labels(n, V, rng, ignored=ignored)
    logp = oracle.token_logprobs(_np(z), y, np.zeros(n))[0]
    ratio = np.exp(0.4 * rng.standard_normal(n))
    for edge in (0.8, 1.3):  # the gradient jumps at the clip's edges: keep off them
        ratio = np.where(np.abs(ratio - edge) < 0.01, edge + 0.02, ratio)
    old = (logp - np.log(ratio)).astype(np.float32)
    adv = rng.standard_normal(n).astype(np.float32)
    ref = (logp + 0.3 * rng.standard_normal(n)).astype(np.float32)
    w = rng.random(n).astype(np.float32)
    w[rng.random(n) < 0.2] = 0.0
    return z, y, yd, old, adv, ref, w


def _cuda(*arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


@gpu
@pytest.mark.parametrize("n,V,dtype,layout", STREAM)
def test_policy_loss_streamed(n, V, dtype, layout):
    test_policy_loss(n, V, layout, dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,V", SIZES)
def test_policy_loss(n, V, layout, dtype):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n * V)
    z, y, yd, old, adv, ref, w = _policy_inputs(n, V, dtype, layout, rng, V + 1, n // 4)
    for kl, ent, weights in ((0.0, 0.0, None), (0.1, 0.0, w), (0.05, 0.02, w)):
        want = oracle.policy_loss(_np(z), y, old, adv, ref if kl else None, weights, 0.2, 0.3, kl, ent)
        o, a, r, wd = _cuda(old, adv, ref if kl else None, weights)
        loss, logps, H, d = kdn.policy_loss_and_grad(z, yd, o, a, ref_logps=r, weights=wd, clip_low=0.2, clip_high=0.3,
                                                     kl_coef=kl, entropy_coef=ent)
        eps = _eps(z, 1.0)
        ww = np.where(y == -100, 0.0, np.full(n, 1.0 / max(1, (y != -100).sum())) if weights is None else w)
        # slope of each term in logp: r |A| <= 4 |A|, kl e^g; the entropy's error is eps (2 + log V)
        coef = ww * (4 * np.abs(adv) + 3 * kl + ent * (2 + np.log(V + 1)) + 1e-30)
        assert np.abs(_np(logps) - want[1]).max() <= eps
        assert np.abs(_np(H) - want[2]).max() <= eps * (2 + np.log(V + 1))
        assert abs(float(loss) - want[0]) <= eps * coef.sum() + 2.0 ** -23 * abs(want[0])
        _assert_grad(d, want[3], coef, eps, dtype)
        plain = kdn.policy_loss(z, yd, o, a, ref_logps=r, weights=wd, clip_low=0.2, clip_high=0.3, kl_coef=kl,
                                entropy_coef=ent)
        assert torch.equal(plain[0], loss) and torch.equal(plain[1], logps) and torch.equal(plain[2], H)


@gpu
def test_policy_loss_autograd_scales_and_refuses_a_second_backward():
    import kdn_b200 as kdn

    rng = np.random.default_rng(5)
    z, y, yd, old, adv, ref, w = _policy_inputs(12, 777, torch.float32, "packed", rng, 9, 2)
    o, a, r = _cuda(old, adv, ref)
    d = kdn.policy_loss_and_grad(z, yd, o, a, ref_logps=r, kl_coef=0.1)[3]
    zg = z.clone().requires_grad_()
    loss, logps, H = kdn.policy_loss(zg, yd, o, a, ref_logps=r, kl_coef=0.1)
    assert loss.requires_grad and not logps.requires_grad and not H.requires_grad
    loss.backward(retain_graph=True)
    assert torch.equal(zg.grad, d)
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    zg.grad = None
    (0.5 * kdn.policy_loss(zg, yd, o, a, ref_logps=r, kl_coef=0.1)[0]).backward()
    assert torch.equal(zg.grad, 0.5 * d)
    three = z.view(3, 4, 777)
    loss3, logps3, _, d3 = kdn.policy_loss_and_grad(three, yd.view(3, 4), o.view(3, 4), a.view(3, 4),
                                                    ref_logps=r.view(3, 4), kl_coef=0.1)
    assert torch.equal(loss3, loss.detach()) and logps3.shape == (3, 4) and torch.equal(d3.view(12, 777), d)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_weight_zero_hold_anything(dtype):
    import kdn_b200 as kdn

    rng = np.random.default_rng(6)
    z, y, yd, old, adv, ref, w = _policy_inputs(6, 300, dtype, "packed", rng, 4, 0)
    w[:] = 0.3
    w[[1, 4]] = 0.0
    o, a, r, wd = _cuda(old, adv, ref, w)
    clean = kdn.policy_loss_and_grad(z, yd, o, a, ref_logps=r, weights=wd, kl_coef=0.1, entropy_coef=0.1)
    z = z.clone()
    z[1], o[4], a[4] = float("nan"), float("inf"), float("nan")
    dirty = kdn.policy_loss_and_grad(z, yd, o, a, ref_logps=r, weights=wd, kl_coef=0.1, entropy_coef=0.1)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[3], dirty[3])
    assert (dirty[3][[1, 4]] == 0).all()
    none = torch.full_like(yd, -100)  # no row counts: the loss is zero, not 0 / 0
    loss, logps, H, d = kdn.policy_loss_and_grad(z, none, o, a)
    assert float(loss) == 0 and not logps.any() and not H.any() and not d.any()
    loss, _, _, d = kdn.policy_loss_and_grad(z[:0], yd[:0], o[:0], a[:0])
    assert float(loss) == 0 and d.shape == (0, 300)


# ------------------------------------------------------------------------------------------------- preference loss
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,V", SIZES)
def test_preference_loss(n, V, layout, dtype):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + 7 * V)
    z = _logits(n, V, dtype, layout, seed=V + 2)
    y, yd = _labels(n, V, rng, [torch.int64, torch.int32][V % 2], ignored=n // 4)
    ref = (oracle.token_logprobs(_np(z), y, np.zeros(n))[0] + 0.2 * rng.standard_normal(n)).astype(np.float32)
    for pairs, use_ref, beta, eps_l, norm in ((1, True, 0.1, 0.0, False), (3, False, 2.0, 0.1, True)):
        cu = np.concatenate([[0], np.sort(rng.integers(0, n + 1, 2 * pairs - 1)), [n]])
        want = oracle.preference_loss(_np(z), y, cu, ref if use_ref else None, beta, eps_l, norm)
        loss, ratios, logps, d = kdn.preference_loss_and_grad(
            z, yd, torch.from_numpy(cu).cuda(), torch.from_numpy(ref).cuda() if use_ref else None, beta=beta,
            label_smoothing=eps_l, length_normalised=norm)
        eps = _eps(z, 1.0)
        longest = 1 if norm else max(1, int(np.diff(cu).max()))
        assert np.abs(_np(logps) - want[2]).max() <= eps
        assert np.abs(_np(ratios) - want[1]).max() <= eps * longest + 2.0 ** -23 * np.abs(want[1]).max()
        assert abs(float(loss) - want[0]) <= 2 * beta * eps * longest + 2.0 ** -23 * abs(want[0])
        # d loss / d logp <= beta / pairs, and moves by beta / pairs x 2 beta eps longest with the log ratios
        _assert_grad(d, want[3], np.full(n, beta / pairs * (1 + 2 * beta * longest)), eps, dtype)
        plain = kdn.preference_loss(z, yd, torch.from_numpy(cu).cuda().int(),
                                    torch.from_numpy(ref).cuda() if use_ref else None, beta=beta,
                                    label_smoothing=eps_l, length_normalised=norm)
        assert torch.equal(plain[0], loss) and torch.equal(plain[1], ratios) and torch.equal(plain[2], logps)


@gpu
def test_preference_loss_edges():
    """Empty sequences have log ratio 0; rows outside every sequence get no gradient; far pairs saturate without
    overflow; the autograd form scales."""
    import kdn_b200 as kdn

    z = _logits(10, 500, torch.float32, "packed", seed=8)
    y = torch.arange(10, device="cuda")
    cu = torch.tensor([2, 5, 5, 5, 8], device="cuda")  # rows 0, 1, 8, 9 outside; sequences 1 and 2 empty
    loss, ratios, logps, d = kdn.preference_loss_and_grad(z, y, cu, beta=0.2)
    assert float(ratios[1]) == 0 and float(ratios[2]) == 0
    assert (d[[0, 1, 8, 9]] == 0).all() and all((d[i] != 0).any() for i in range(2, 8))
    zg = z.clone().requires_grad_()
    (3.0 * kdn.preference_loss(zg, y, cu, beta=0.2)[0]).backward()
    assert torch.equal(zg.grad, 3.0 * d)
    far = torch.zeros(2, 4, device="cuda")
    far[0, 0], far[1, 0] = 3000.0, -3000.0
    two = torch.tensor([0, 1, 2], device="cuda")
    first = torch.zeros(2, dtype=torch.int64, device="cuda")
    loss, ratios, _, d = kdn.preference_loss_and_grad(far, first, two, beta=1.0)
    assert float(loss) == 0.0 and not d.any()
    loss, ratios, _, d = kdn.preference_loss_and_grad(far.flip(0).contiguous(), first, two, beta=1.0)
    assert abs(float(loss) - (3000.0 + float(np.log(3)))) < 1e-2 and torch.isfinite(d).all()
    loss, ratios, logps, d = kdn.preference_loss_and_grad(z[:0], y[:0], torch.tensor([0, 0, 0], device="cuda"))
    assert abs(float(loss) - np.log(2)) < 1e-6 and not ratios.any() and d.shape == (0, 500)


# ----------------------------------------------------------------------------------------------- distillation loss
def _teacher(n, V, K, rng, T, dtype=np.float32):
    ids = np.stack([rng.permutation(V)[:K] for _ in range(n)])
    t = np.sort(2.5 * rng.standard_normal((n, K)) + 4, axis=1)[:, ::-1].astype(dtype)
    m = (t / T).max(-1)
    lse = m + np.log(np.exp(t / T - m[:, None]).sum(-1)) - np.log(0.6 + 0.35 * rng.random(n))
    return ids, t, lse.astype(np.float32)


@gpu
@pytest.mark.parametrize("n,V,dtype,layout,K", [(*c, k) for c, k in zip(STREAM, (1, 128, 33, 64, 100, 7))])
def test_distillation_loss_streamed(n, V, dtype, layout, K):
    test_distillation_loss(n, V, K, layout, dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_streamed_rows_with_infinities_and_repeated_ids(dtype):
    """The masks of the other tests in rows that are streamed: -inf, nothing left, NaN, ignored rows that hold NaN, the
    type's lowest value, ids given twice, a masked id."""
    import kdn_b200 as kdn

    n, V, K, inf = 300, 20000, 40, float("inf")
    rng = np.random.default_rng(12)
    z = _logits(n, V, dtype, "packed", seed=21).clone()
    z[0, 1::2], z[1], z[2, 77], z[3] = -inf, -inf, float("nan"), float("nan")
    z[4] = torch.finfo(dtype).min
    z[5, 1:] = -inf
    y, yd = _labels(n, V, rng, ignored=0)
    y[:6] = [0, 0, 5, -100, 9, 0]
    yd = torch.from_numpy(y).cuda()
    old, adv = -9 - rng.random(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    w = (rng.random(n) / n).astype(np.float32)
    want = oracle.policy_loss(_np(z), y, old, adv, None, w, 0.2, 0.2, 0.0, 0.01)
    o, a, wd = _cuda(old, adv, w)
    loss, logps, H, d = kdn.policy_loss_and_grad(z, yd, o, a, weights=wd, entropy_coef=0.01)
    fine = [i for i in range(n) if i not in (1, 2)]
    eps = 2.0 ** -23 * 60 + 2.0 ** -17
    assert np.isnan(_np(logps)[[1, 2]]).all() and np.isnan(_np(d)[[1, 2]]).all() and torch.isnan(loss)
    assert np.abs(_np(logps) - want[1])[fine].max() <= eps
    assert np.abs(_np(H) - want[2])[fine].max() <= eps * (2 + np.log(V))
    ratio = np.exp(np.clip(want[1] - old, -30, 3))
    coef = w * (np.abs(adv) * (1 + ratio) + 0.01 * (2 + np.log(V))) + 1e-30
    _assert_grad(d[fine], want[3][fine], coef[fine], eps, dtype)
    assert not d[3].any()
    for tail in (False, True):
        ids, t, lse = _teacher(n, V, K, rng, 1.0)
        ids[6, 5] = ids[6, 9] = ids[6, 1]
        ids[7, :] = V + 1
        ids[3, 0] = -1
        z[8, ids[8, 2]] = -inf
        lse = (np.log(np.exp(t.astype(np.float64)).sum(-1)) + 0.3).astype(np.float32)
        want = oracle.distillation_loss(_np(z), t, ids, lse if tail else None, w)
        td, idd, ld = _cuda(t, ids, lse if tail else None)
        loss, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd)
        got = _np(kl)
        assert np.isnan(got[[1, 2]]).all() and got[3] == 0 and got[7] == 0 and got[8] == inf
        rows = [i for i in range(n) if i not in (0, 1, 2, 5, 8)]
        assert np.abs(got - want[1])[rows].max() <= 30 * (eps + 2.0 ** -23 * 40)
        assert not d[3].any() and not d[7].any()
        _assert_grad(d[rows], want[2][rows], 21 * w[rows], eps + 2.0 ** -23 * 40, dtype)
    import ctypes

    from kdn_b200 import _lib
    code = ctypes.c_int(0)
    assert _lib.load().kdn_device_error(_lib.stream_handle(z.device), ctypes.byref(code)) == 0 and code.value == 1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,V,K", [(3, 2, 1), (5, 7, 3), (33, 200, 40), (9, 4099, 64), (200, 4096, 17), (7, 32000, 64),
                                   (2, 50021, 1024), (3, 131072, 100), (1, 262145, 5), (2, 300007, 256)])
def test_distillation_loss(n, V, K, layout, dtype):
    import kdn_b200 as kdn

    rng = np.random.default_rng(n + V + K)
    T = [1.0, 2.0][(n + K) % 2]
    z = _logits(n, V, dtype, layout, seed=V + 3)
    ids, t, lse = _teacher(n, V, K, rng, T)
    ids[rng.random((n, K)) < 0.1] = -1
    ids[:, 0] = np.where(ids[:, 0] < 0, rng.integers(0, V, n), ids[:, 0])
    ids[n // 2, 0] = -1 if n > 2 else ids[n // 2, 0]
    w = rng.random(n).astype(np.float32)
    w[rng.random(n) < 0.2] = 0.0
    for tail, weights in ((False, None), (True, w)):
        want = oracle.distillation_loss(_np(z), t, ids, lse if tail else None, weights, T)
        td, idd, ld, wd = _cuda(t, ids.astype([np.int64, np.int32][K % 2]), lse if tail else None, weights)
        loss, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd, temperature=T)
        eps = _eps(z, T) + 2.0 ** -23 * (np.abs(t).max() / T + 20)
        live = ids[:, 0] >= 0
        ww = np.where(live, np.full(n, 1.0 / max(1, live.sum())) if weights is None else w, 0.0)
        # p_rest = 1 - sum p is within eps absolutely, log(p_rest / q_rest) within eps / p_rest (p_rest >= 0.05)
        assert np.abs(_np(kl) - want[1]).max() <= (30 if tail else 2) * eps
        assert abs(float(loss) - want[0]) <= T * T * ww.sum() * (30 if tail else 2) * eps + 2.0 ** -23 * abs(want[0])
        rest_ratio = 1.0  # p_rest / q_rest scales the error of q outside the ids; both are below one
        _assert_grad(d, want[2], ww * T * (1 + (20 if tail else 0) * rest_ratio), eps, dtype)
        plain = kdn.distillation_loss(z, td, idd, teacher_lse=ld, weights=wd, temperature=T)
        assert torch.equal(plain[0], loss) and torch.equal(plain[1], kl)
        again = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd, temperature=T)
        assert torch.equal(again[0], loss) and torch.equal(again[2], d)


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_edges(dtype, tail):
    """Ids given twice count twice; -inf teacher entries weigh nothing; rows without an id, of weight zero or whose
    only ids lie outside the vocabulary give zeros whatever they hold; a masked student entry gives an infinite
    divergence; teacher logits in bf16."""
    import kdn_b200 as kdn

    V, K = 700, 6
    rng = np.random.default_rng(1)
    z = _logits(7, V, dtype, "packed", seed=5).clone()
    ids, t, lse = _teacher(7, V, K, rng, 1.0)
    ids[0, 3] = ids[0, 1]                       # twice
    ids[1, 2:] = ids[1, 1]                      # five times
    t[2, 4] = -np.inf                           # a teacher entry of no weight
    ids[3, 0] = -1                              # ignored
    z[3] = float("nan")
    z[4] = float("nan")                         # weight zero
    ids[5, :] = V + 3                           # nothing valid
    z[6, ids[6, 2]] = -float("inf")             # masked in the student
    lse = (np.log(np.exp(np.where(ids >= 0, t, -np.inf).astype(np.float64)).sum(-1)) + 0.3).astype(np.float32)
    w = np.array([0.2, 0.3, 0.1, 0.4, 0.0, 0.5, 0.1], np.float32)
    want = oracle.distillation_loss(_np(z), t, ids, lse if tail else None, w)
    td, idd, ld, wd = _cuda(t, ids, lse if tail else None, w)
    loss, kl, d = kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd)
    got, eps = _np(kl), _eps(z[:3], 1.0) + 2.0 ** -23 * 40
    assert (np.abs(got[:3] - want[1][:3]) <= 30 * eps).all()
    assert got[3] == 0 and got[5] == 0 and got[6] == np.inf and float(loss) == np.inf
    g = _np(d)
    assert (g[3] == 0).all() and (g[4] == 0).all() and (g[5] == 0).all()
    rows = [0, 1, 2, 6]
    _assert_grad(d[rows], want[2][rows], (20 * w)[rows], eps, dtype)
    import ctypes
    from kdn_b200 import _lib
    code = ctypes.c_int(0)
    assert _lib.load().kdn_device_error(_lib.stream_handle(z.device), ctypes.byref(code)) == 0 and code.value == 1
    tb = td[:1].bfloat16()
    a = kdn.distillation_loss(z[:1], tb, idd[:1])
    b = kdn.distillation_loss(z[:1], tb.float(), idd[:1])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    zg = z[:3].clone().requires_grad_()
    (2.0 * kdn.distillation_loss(zg, td[:3], idd[:3], weights=wd[:3])[0]).backward()
    assert torch.equal(zg.grad, 2.0 * kdn.distillation_loss_and_grad(z[:3], td[:3], idd[:3], weights=wd[:3])[2])


# --------------------------------------------------------------------------------------- gradients by differences
@gpu
def test_gradients_against_differences():
    """Directional derivatives of the float64 losses by central differences, against the kernels' gradients."""
    import kdn_b200 as kdn

    rng = np.random.default_rng(11)
    n, V, K = 14, 1234, 20
    z, y, yd, old, adv, ref, w = _policy_inputs(n, V, torch.float32, "packed", rng, 3, 2)
    o, a, r, wd = _cuda(old, adv, ref, w)
    ids, t, lse = _teacher(n, V, K, rng, 1.5)
    td, idd, ld = _cuda(t, ids, lse)
    cu = np.array([0, 4, 7, 12, 14])
    z64 = _np(z)
    pairs = [
        (lambda x: oracle.policy_loss(x, y, old, adv, ref, w, 0.2, 0.3, 0.1, 0.05)[0],
         kdn.policy_loss_and_grad(z, yd, o, a, ref_logps=r, weights=wd, clip_low=0.2, clip_high=0.3, kl_coef=0.1,
                                  entropy_coef=0.05)[-1]),
        (lambda x: oracle.preference_loss(x, y, cu, ref, 0.3, 0.1)[0],
         kdn.preference_loss_and_grad(z, yd, torch.from_numpy(cu).cuda(), r, beta=0.3, label_smoothing=0.1)[-1]),
        (lambda x: oracle.distillation_loss(x, t, ids, None, w, 1.5)[0],
         kdn.distillation_loss_and_grad(z, td, idd, weights=wd, temperature=1.5)[-1]),
        (lambda x: oracle.distillation_loss(x, t, ids, lse, w, 1.5)[0],
         kdn.distillation_loss_and_grad(z, td, idd, teacher_lse=ld, weights=wd, temperature=1.5)[-1]),
    ]
    for f, g in pairs:
        for _ in range(3):
            d = rng.standard_normal((n, V))
            slope = (_np(g) * d).sum()
            # |d| ~ 1 an element and |g| summed over a row at most 2 |coef|: 100 eps in all
            assert abs(_differences(f, z64, d) - slope) <= 100 * _eps(z, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,ld", [(1, 1, 1), (3, 2, 2), (5, 7, 16), (67, 1000, 1000), (2500, 130, 131),
                                    (9, 4099, 4099), (33, 20011, 20016), (3, 70001, 70001)])
def test_gradients_scaled_in_place(n, V, ld, dtype):
    """The factor of an upstream gradient: one product in fp32, rounded once; what lies beside the rows stays."""
    from kdn_b200 import _lib

    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(n + V)
    x = torch.randn(n, ld, device="cuda", generator=gen).to(dtype)
    for factor in (1.0, 2.5, 0.0, -0.125):
        want, got = x.clone(), x.clone()
        want[:, :V] = (x[:, :V].float() * factor).to(dtype)
        scale = torch.tensor(factor, device="cuda")
        assert lib.kdn_scale_rows(got.data_ptr(), _lib.dtype_code(got), ld, n, V, scale.data_ptr(),
                                  torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(got, want), factor


@pytest.mark.gpu
@pytest.mark.parametrize("n,V", [(16, 4100), (600, 32000)])
def test_losses_replayed_from_a_graph(n, V):
    import kdn_b200 as kdn

    gen = torch.Generator(device="cuda").manual_seed(n)
    z = torch.randn(n, V, device="cuda", generator=gen).to(torch.bfloat16)
    y = torch.randint(V, (n,), device="cuda", generator=gen)
    old, adv = (torch.randn(n, device="cuda", generator=gen) for _ in range(2))
    ids = torch.randint(V, (n, 33), device="cuda", generator=gen)
    top = torch.randn(n, 33, device="cuda", generator=gen)
    cu = torch.tensor([0, n // 4, n // 2, n // 2 + 3, n], device="cuda")
    calls = [lambda: (kdn.token_logprobs(z, y),), lambda: kdn.policy_loss_and_grad(z, y, old, adv, ref_logps=old),
             lambda: kdn.preference_loss_and_grad(z, y, cu), lambda: kdn.distillation_loss_and_grad(z, top, ids)]
    for call in calls:
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for _ in range(2):
            for t in got:
                t.fill_(-1)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(want, got))
