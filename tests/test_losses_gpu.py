"""The losses over vocabulary logits (token log-probabilities, preference, clipped
policy, distillation) and their gradients against their formulas in fp64.

Tolerances. u = 2^-24. An exponential 2^((x - max) c) carries the fp32 roundings of the
difference, of c and of the product (3 u of the exponent a, so 3 u a ln 2 of the value)
and ex2.approx's 2^-22: relative 4 u + 2.1 u a. In the row's sum the exponents
average at most log2 V (the entropy bound), and V / 512 + 16 additions round once each:
    rel_s = (4 + 2.1 log2 V + V / 512 + 16) u
which is the absolute error of a log-probability before its own rounding, u |lp|.
A probability has rel_q = rel_s + (4 + 2.1 a_max) u. A gradient k (onehot - q) then
is off by |k| q rel_q + 8 u |k (onehot - q)| + 2 u |k| onehot, and by half a step of its type.
Losses move with the log-probabilities by at most sum |dloss/dlp| times their error."""
import math

import pytest
import torch

from lema_b200 import _native, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
IGN = -100


def rel_s(V):
    return (20 + 2.1 * math.log2(max(V, 2)) + V / 512) * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(dev, B, S, V, dtype, seed=0, ignore=0.3):
    g = torch.Generator(device=dev).manual_seed(seed + 7 * V + S)
    x = (torch.randn(B, S, V, device=dev, generator=g) * 2).to(DT[dtype])
    t = torch.randint(0, V, (B, S), device=dev, generator=g)
    up = torch.rand(B, S, 1, device=dev, generator=g) * 8
    x.scatter_(-1, t[..., None], (x.gather(-1, t[..., None]).float() + up).to(x.dtype))
    if ignore:
        t[torch.rand(B, S, device=dev, generator=g) < ignore] = IGN
    return x, t, g


def ref_logps(x, t, tau=1.0):
    """fp64 log-probabilities (0 where ignored) and probabilities of every row."""
    z = x.double() / tau
    lsm = torch.log_softmax(z, -1)
    lp = lsm.gather(-1, t.clamp(min=0)[..., None])[..., 0]
    return torch.where(t == IGN, torch.zeros_like(lp), lp), lsm.exp()


def check_logps(got, want, V):
    assert got.dtype == torch.float32
    err = (got.double() - want).abs()
    assert (err <= rel_s(V) + U * want.abs()).all(), err.max().item()


def check_dx(got, x, q, k, mass, tau=1.0, mass_err=2 * U):
    """got = k (mass - q): k [rows] fp64, mass the row's point masses."""
    k = k[..., None]
    want = k * (mass - q)
    a_max = (x.double().amax(-1) - torch.where(x.isinf(), 0.0, x.double()).amin(-1)).max().item() \
        / tau * 1.4427
    rel_q = rel_s(x.shape[-1]) + (4 + 2.1 * min(a_max, 150.0)) * U
    tol = ((half_step(got.dtype) + 8 * U) * want.abs()
           + k.abs() * (q * rel_q + mass_err * mass) + 1e-37)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


def onehot(t, V):
    m = torch.zeros(*t.shape, V, dtype=torch.float64, device=t.device)
    m.scatter_(-1, t.clamp(min=0)[..., None], 1.0)
    return torch.where((t == IGN)[..., None], 0.0, m)


SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (1, 5, 31), (3, 17, 512), (2, 9, 4097), (2, 5, 32000),
          (1, 7, 32768), (1, 3, 32776), (2, 2, 50257), (1, 3, 65544), (1, 2, 128256),
          (1, 1, 151937), (1, 2, 262144), (1, 1, 300001), (40, 64, 130), (300, 1, 1000)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S,V", SHAPES)
def test_token_logprobs(cuda_device, B, S, V, dtype):
    for tau in (1.0, 0.7):
        x, t, g = make(cuda_device, B, S, V, dtype)
        if B * S > 1:
            t.view(-1)[0] = V - 1
            t.view(-1)[-1] = 0
        x.requires_grad_(True)
        lp = ops.token_logprobs(x, t, temperature=tau)
        want, q = ref_logps(x.detach(), t, tau)
        check_logps(lp.detach(), want, V)
        assert torch.equal(ops.token_logprobs(x.detach(), t, temperature=tau), lp.detach())
        up = torch.randn(B, S, device=cuda_device, generator=g)
        (dx,) = torch.autograd.grad(lp, x, up)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        k = torch.where(t == IGN, 0.0, up.double() / tau)
        check_dx(dx, x.detach(), q, k, onehot(t, V), tau)


def _layouts(dev, dtype):
    x, t, _ = make(dev, 3, 12, 1000, dtype)
    big = torch.zeros(3, 12, 1100, dtype=x.dtype, device=dev)
    for off in (0, 1, 8):
        view = big.clone()[:, :, off:off + 1000]
        view.copy_(x)
        yield f"rows of a wider buffer, offset {off}", view, t
    yield "without the last position", x[:, :-1], t[:, :-1]
    yield "every second position", x[:, ::2], t[:, ::2]
    yield "positions outermost", x.transpose(0, 1).contiguous().transpose(0, 1), t
    yield "vocabulary outermost", x.permute(2, 0, 1).contiguous().permute(1, 2, 0), t
    yield "one row for all", x[:1, :1].expand(3, 12, 1000), t
    yield "two-dimensional", x.view(36, 1000), t.view(36)
    yield "four-dimensional", x.view(3, 4, 3, 1000), t.view(3, 4, 3)
    yield "four-dimensional, permuted", x.view(3, 4, 3, 1000).transpose(1, 2), \
        t.view(3, 4, 3).transpose(1, 2)
    odd = torch.zeros(3 * 12 * 1000 + 3, dtype=x.dtype, device=dev)[3:].view(3, 12, 1000)
    odd.copy_(x)
    yield "base off by three elements", odd, t


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layouts(cuda_device, dtype):
    for name, x, t in _layouts(cuda_device, dtype):
        want, q = ref_logps(x, t)
        x = x.detach().requires_grad_(True)
        lp = ops.token_logprobs(x, t)
        check_logps(lp.detach(), want, 1000)
        (dx,) = torch.autograd.grad(lp.sum(), x)
        check_dx(dx, x.detach(), q, torch.where(t == IGN, 0.0, 1.0).double(), onehot(t, 1000))
        adv = torch.ones_like(want, dtype=torch.float32)
        loss, lps, _, dx2 = ops.policy_loss_grad(x.detach(), t, None, adv)
        n = (t != IGN).sum().double()
        check_logps(lps, want, 1000)
        check_dx(dx2, x.detach(), q, torch.where(t == IGN, 0.0, -1.0).double() / n, onehot(t, 1000))
        assert abs(loss.item() + 1.0) <= 2 * U, name


def test_ignored_rows_are_not_read(cuda_device):
    for dtype in DT:
        x, t, _ = make(cuda_device, 2, 24, 5000, dtype, ignore=0.5)
        clean = ops.preference_loss_grad(x, t)
        x2 = x.clone()
        x2[t == IGN] = float("nan")
        ref = torch.where(t == IGN, float("nan"), 0.0)
        for a, b in zip(clean, ops.preference_loss_grad(x2, t, ref)):
            assert torch.equal(a, b)
        assert (clean[2][t == IGN] == 0).all()
        adv = torch.where(t == IGN, float("inf"), 1.5)
        old = torch.where(t == IGN, float("nan"), ops.token_logprobs(x, t))
        loss, lps, kl, dx = ops.policy_loss_grad(x2, t, old, adv, ref)
        assert torch.isfinite(loss) and torch.isfinite(kl) and torch.isfinite(dx.float()).all()
        assert (lps[t == IGN] == 0).all() and (dx[t == IGN] == 0).all()
        ids = torch.zeros(2, 24, 3, dtype=torch.int64, device=cuda_device)
        ids[t == IGN] = 10 ** 12
        tl = torch.where((t == IGN)[..., None], float("nan"), 1.0).expand(2, 24, 3)
        loss, dx = ops.distill_loss_grad(x2, ids, tl, t != IGN)
        assert torch.isfinite(loss) and (dx[t == IGN] == 0).all()


@pytest.mark.parametrize("V", [130, 9001])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_infinities_and_lowest_values(cuda_device, dtype, V):
    low = torch.finfo(DT[dtype]).min
    x, t, _ = make(cuda_device, 1, 8, V, dtype, ignore=0)
    t[:] = 3
    x[0, 0, 10:] = float("-inf")         # most of the vocabulary masked
    x[0, 1, :] = low                     # masked whole by the lowest value: uniform
    x[0, 2, :] = low
    x[0, 2, 3] = 0.0                     # one token left
    x[0, 3, 3] = float("-inf")           # the target itself masked
    x[0, 4, :] = float("-inf")           # nothing left: NaN, as log_softmax gives
    x[0, 5, 7] = float("nan")
    x[0, 6, 5] = float("inf")
    for tau in (1.0, 0.5):
        xr = x.clone().requires_grad_(True)
        lp = ops.token_logprobs(xr, t, temperature=tau)
        # lowest values overflow when divided by a temperature below 1: subtract the maximum first
        z = x.double()
        z = torch.log_softmax((z - z.amax(-1, keepdim=True)) / tau, -1)
        want = z[..., 3]
        got = lp.detach().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        assert want.isnan().tolist()[0] == [False] * 4 + [True] * 3 + [False]
        ok = torch.isfinite(want)
        assert ((got - want).abs()[ok] <= (rel_s(V) + U * want.abs())[ok]).all()
        (dx,) = torch.autograd.grad(lp, xr, torch.ones_like(lp))
        assert dx[0, 4:7].isnan().all()
        for r in (0, 1, 2, 3, 7):
            q = z[0, r].exp()
            mass = torch.zeros_like(q)
            mass[3] = 1
            err = (dx[0, r].double() - (mass - q) / tau).abs()
            tol = (half_step(x.dtype) + 8 * U) * (mass - q).abs() / tau \
                + (q * (rel_s(V) + 300 * U) + 2 * U * mass) / tau + 1e-37
            assert (err <= tol).all(), (r, err.max())


def ref_preference(x, t, ref, beta, e):
    lp, q = ref_logps(x, t)
    keep = (t != IGN)
    d = torch.where(keep, lp - (0 if ref is None else ref.double()), 0.0)
    P = x.shape[0] // 2
    R = beta * d.sum(1)
    h = R[:P] - R[P:]
    sp = torch.nn.functional.softplus
    loss = ((1 - e) * sp(-h) + e * sp(h)).mean()
    dh = (e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h)) * beta / P
    k = torch.cat([dh, -dh])[:, None] * keep
    return loss, R, k, q


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("P,S,V,beta,e", [(1, 1, 5, 0.1, 0.0), (1, 40, 1000, 0.1, 0.1),
                                          (3, 33, 4099, 0.5, 0.0), (2, 70, 32000, 0.1, 0.2),
                                          (1, 5, 128256, 5.0, 0.0), (160, 2, 300, 0.3, 0.1)])
def test_preference(cuda_device, P, S, V, beta, e, dtype):
    x, t, g = make(cuda_device, 2 * P, S, V, dtype)
    if S > 1:
        t[0, :] = IGN                    # a chosen sequence without a counted token
    lp, _ = ref_logps(x, t)
    refs = [None, (lp + torch.randn(lp.shape, device=x.device, generator=g,
                                    dtype=torch.float64) * 0.2).float()]
    for ref in refs:
        loss, rewards, dx = ops.preference_loss_grad(x, t, ref, beta=beta, label_smoothing=e)
        want, R, k, q = ref_preference(x, t, ref, beta, e)
        n = (t != IGN).sum(1)
        lp_err = rel_s(V) + U * lp.abs().amax(1)      # the log-probabilities pass through fp32
        r_err = beta * n * lp_err
        assert ((rewards.double() - R).abs() <= r_err + U * R.abs() + 1e-30).all()
        h_err = (r_err[:P] + r_err[P:])
        assert abs(loss.item() - want.item()) <= h_err.mean() + 2 * U * abs(want.item())
        # sigma moves by at most its value times the error of h
        slack = 1 + 2 * torch.cat([h_err, h_err])[:, None]
        for scale in (1.0, 0.25):
            got = dx if scale == 1.0 else ops.preference_loss_grad(
                x, t, ref, beta=beta, label_smoothing=e, grad_scale=scale)[2]
            a = k * scale
            mass = onehot(t, V)
            wantx = a[..., None] * (mass - q)
            tol = (half_step(x.dtype) + 8 * U) * wantx.abs() \
                + a.abs()[..., None] * (q * (rel_s(V) + 90 * U) + 2 * U * mass) \
                + (slack - 1)[..., None] * (k.abs().amax() * scale) * (mass - q).abs() + 1e-37
            assert ((got.double() - wantx).abs() <= tol).all()
        xr = x.clone().requires_grad_(True)
        l2, rw2 = ops.preference_loss(xr, t, ref, beta=beta, label_smoothing=e)
        assert torch.equal(l2.detach(), loss) and torch.equal(rw2, rewards)
        assert not rw2.requires_grad
        (gx,) = torch.autograd.grad(l2, xr, torch.tensor(1.0, device=x.device))
        assert torch.equal(gx, dx)


def ref_policy(x, t, old, adv, ref, clip, kl_coef, tau, reduction):
    lp, q = ref_logps(x, t, tau)
    keep = t != IGN
    A = adv.double() if adv.dim() == t.dim() else adv.double()[:, None].expand(t.shape)
    n = keep.sum() if reduction == "token" else t.shape[0] * keep.sum(-1, keepdim=True)
    w = torch.where(keep, 1.0 / n.clamp(min=1).double(), 0.0)
    r = torch.exp(lp - old.double()) if old is not None else torch.ones_like(lp)
    bent = r.clamp(1 - clip[0], 1 + clip[1])
    surr = -torch.minimum(r * A, bent * A)
    k = torch.where(r * A <= bent * A, -r * A, 0.0)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref.double() - lp
        kl = torch.expm1(d) - d
        k = k - kl_coef * torch.expm1(d)
    return (w * (surr + kl_coef * kl)).sum(), lp, (w * kl).sum(), w * k, q


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S,V,tau,kl,reduction", [
    (1, 1, 4, 1.0, 0.0, "token"), (3, 29, 777, 1.0, 0.1, "token"),
    (4, 31, 4096, 0.8, 0.05, "sequence"), (2, 40, 32000, 1.0, 0.0, "token"),
    (2, 6, 100277, 1.3, 0.2, "sequence"), (200, 3, 128, 1.0, 0.04, "sequence")])
def test_policy(cuda_device, B, S, V, tau, kl, reduction, dtype):
    x, t, g = make(cuda_device, B, S, V, dtype)
    if B > 1:
        t[1, :] = IGN                    # a sequence without a counted token
    lp, _ = ref_logps(x, t, tau)
    clip = (0.2, 0.3)
    d = torch.randn(B, S, device=x.device, generator=g, dtype=torch.float64) * 0.2
    for edge in (math.log(0.8), math.log(1.3)):   # the gradient jumps there
        d = torch.where((d - edge).abs() < 1e-3, edge + 2e-3, d)
    old = (lp - d).float()
    ref = (lp + torch.randn(B, S, device=x.device, generator=g, dtype=torch.float64) * 0.3).float()
    adv2 = torch.randn(B, S, device=x.device, generator=g)
    adv1 = torch.randn(B, device=x.device, generator=g)
    for o, adv, r in ((old, adv2, ref), (old, adv1, None), (None, adv1, ref)):
        kw = dict(clip=clip, kl_coef=kl, temperature=tau, reduction=reduction)
        loss, lps, klv, dx = ops.policy_loss_grad(x, t, o, adv, r, **kw)
        want, wlp, wkl, k, q = ref_policy(x, t, o, adv, r, clip, kl, tau, reduction)
        check_logps(lps, wlp, V)
        # per token: |d loss / d lp| <= |coef|, second order below; kl's slope is |e^d - 1|
        e_lp = rel_s(V)
        s_abs = ref_policy(x, t, o, adv.abs(), r, (1.0, 1e6), kl, tau, reduction)
        bound = 4 * e_lp * (s_abs[3].abs().sum() + 1e-3) + 2 * U * abs(want.item()) \
            + 4 * U * s_abs[0].abs()
        assert abs(loss.item() - want.item()) <= bound
        assert abs(klv.item() - wkl.item()) <= bound + 2 * e_lp
        a_max = (x.double().amax(-1) - x.double().amin(-1)).max().item() / tau * 1.4427
        rel_q = rel_s(V) + (4 + 2.1 * a_max) * U
        mass = onehot(t, V)
        kk = (k / tau)[..., None]
        # a coefficient moves by its token's |A| r + kl e^d times the log-probability's error
        wobble = 4 * e_lp * (torch.where(t == IGN, 0.0, 1.0).double() * 4 * (adv.abs().max() + kl)
                             / (tau * max(1, int((t != IGN).sum()) if reduction == "token"
                                          else B)))[..., None]
        wantx = kk * (mass - q)
        tol = (half_step(x.dtype) + 8 * U) * wantx.abs() + (kk.abs() + wobble) * (q * rel_q) \
            + wobble * (mass - q).abs() + 2 * U * kk.abs() * mass + 1e-37
        assert ((dx.double() - wantx).abs() <= tol).all()
        xr = x.clone().requires_grad_(True)
        l2, lp2, kl2 = ops.policy_loss(xr, t, o, adv, r, **kw)
        assert torch.equal(l2.detach(), loss) and torch.equal(lp2, lps) and torch.equal(kl2, klv)
        (g1,) = torch.autograd.grad(l2, xr, torch.tensor(0.5, device=x.device))
        err = (g1.double() - 0.5 * wantx).abs()
        assert (err <= 0.5 * tol + 1e-37).all()


def ref_distill(x, ids, tl, mask, tau):
    V = x.shape[-1]
    keep = mask.clone() if mask is not None else torch.ones(x.shape[:-1], dtype=torch.bool,
                                                            device=x.device)
    z = tl.double() / tau
    empty = torch.isinf(tl).all(-1) & (tl < 0).all(-1)
    lt = torch.log_softmax(torch.where(empty[..., None], 0.0, z), -1)
    p = lt.exp() * ~empty[..., None]
    _, q = ref_logps(x, torch.zeros(x.shape[:-1], dtype=torch.int64, device=x.device), tau)
    lq = torch.log_softmax(x.double() / tau, -1).gather(-1, ids.clamp(0, V - 1).long())
    terms = torch.where(p > 0, p * (lt - lq), 0.0).sum(-1)
    n = max(1, int(keep.sum()))
    loss = tau * tau * (terms * keep).sum() / n
    mass = torch.zeros_like(q).scatter_add_(-1, ids.clamp(0, V - 1).long(), p)
    k = (keep & ~empty).double() * (-tau / n)
    return loss, k, mass, q


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S,V,K,tau", [(1, 1, 3, 1, 1.0), (2, 9, 100, 7, 2.0),
                                         (1, 20, 4099, 64, 1.0), (2, 16, 32000, 64, 2.0),
                                         (1, 4, 50257, 1024, 4.0), (1, 2, 128256, 100, 1.0),
                                         (70, 4, 96, 96, 3.0)])
def test_distill(cuda_device, B, S, V, K, tau, dtype):
    x, _, g = make(cuda_device, B, S, V, dtype)
    noisy = x.float() + torch.randn(x.shape, device=x.device, generator=g)
    tl, ids = torch.topk(noisy, min(K, V), -1)
    mask = torch.rand(B, S, device=x.device, generator=g) > 0.3
    mask.view(-1)[0] = True
    cases = [(ids, tl, mask), (ids.int(), tl.bfloat16(), None)]
    if K > 4:
        dup, gone = ids.clone(), tl.clone()
        dup[..., 2] = dup[..., 0]        # an index twice, one three times
        dup[..., 3] = dup[..., 1]
        dup[..., 4] = dup[..., 1]
        gone[..., 5:] = float("-inf")    # short lists: padded with no entries
        bad = dup.clone()
        bad[..., 5:] = -1                # whatever index those hold
        gone.view(-1, gone.shape[-1])[-1] = float("-inf")   # a row without any entry
        cases += [(dup, tl, mask), (bad, gone, None)]
    for i, v, m in cases:
        loss, dx = ops.distill_loss_grad(x, i, v, m, temperature=tau)
        want, k, mass, q = ref_distill(x, i, v, m, tau)
        # weights p are rounded to fp32 once, log q carries rel_s; both enter times tau^2
        assert abs(loss.item() - want.item()) <= tau * tau * (rel_s(V) + 60 * U) \
            + 2 * U * abs(want.item())
        a_max = (x.double().amax(-1) - x.double().amin(-1)).max().item() / tau * 1.4427
        rel_q = rel_s(V) + (4 + 2.1 * a_max) * U
        kk = k[..., None]
        wantx = kk * (mass - q)
        # masses of a repeated index add K roundings
        tol = (half_step(x.dtype) + 8 * U) * wantx.abs() \
            + kk.abs() * (q * rel_q + (4 + K) * U * mass) + 1e-37
        assert ((dx.double() - wantx).abs() <= tol).all()
        xr = x.clone().requires_grad_(True)
        l2 = ops.distill_loss(xr, i, v, m, temperature=tau)
        assert torch.equal(l2.detach(), loss)
        (g1,) = torch.autograd.grad(l2 * 3.0, xr)
        assert ((g1.double() - 3 * wantx).abs() <= 3 * tol).all()


def test_gradients_against_differences(cuda_device):
    """Central differences along a direction d, |d| <= 1: the third derivative of a
    log-probability along it is at most 1 (a third cumulant of a variable in [-1, 1])
    and the second at most 1, the first at most 2; with step e the quotient is off by e^2 / 6 of the
    loss's third derivative and by 2 u |loss| / e."""
    e = 2.0 ** -6
    x, t, g = make(cuda_device, 2, 6, 333, "fp32", ignore=0.2)
    d = torch.rand(x.shape, device=x.device, generator=g) * 2 - 1
    d = (d * 64).round() / 64
    x = (x * 1024).round() / 1024                     # x +- e d is exact
    w = torch.randn(2, 6, device=x.device, generator=g).double()
    old = ops.token_logprobs(x, t)
    adv = torch.randn(2, 6, device=x.device, generator=g)
    tl, ids = torch.topk(x + torch.randn(x.shape, device=x.device, generator=g), 9, -1)
    n = int((t != IGN).sum())

    def lp_sum(v):
        return (ops.token_logprobs(v, t).double() * w).sum()

    def pref(v):
        return ops.preference_loss(v, t, beta=0.05)[0]

    def pol(v):
        return ops.policy_loss(v, t, old, adv, old - 0.1, clip=(1.0, 100.0), kl_coef=0.3)[0]

    def dist(v):
        return ops.distill_loss(v, ids, tl)

    bt = 0.05 * n
    third = {"lp": w.abs().sum().item(),
             "pref": 0.1 * (2 * bt) ** 3 + 3 * 0.25 * 2 * bt * bt + bt,
             "pol": (adv.abs().max().item() * 1.2 + 0.3 * 1.2) * (8 + 6 + 1),
             "dist": 1.0}
    for name, f in (("lp", lp_sum), ("pref", pref), ("pol", pol), ("dist", dist)):
        xr = x.clone().requires_grad_(True)
        loss = f(xr)
        (gx,) = torch.autograd.grad(loss, xr)
        slope = (gx.double() * d.double()).sum().item()
        hi, lo = f(x + e * d).item(), f(x - e * d).item()
        size = max(abs(hi), abs(lo)) if name != "lp" else w.abs().sum().item() * 20
        # the gradient's own fp32 roundings: 60 u of each |entry|
        own = 60 * U * (gx.double() * d.double()).abs().sum().item() + 10 * rel_s(333)
        tol = e * e / 6 * third[name] + (2 * U * size + 2 * rel_s(333) * third[name]) / e + own
        assert abs((hi - lo) / (2 * e) - slope) <= tol, (name, (hi - lo) / (2 * e), slope, tol)


def test_no_counted_row(cuda_device):
    x, t, _ = make(cuda_device, 2, 5, 400, "bf16")
    t[:] = IGN
    loss, lps, kl, dx = ops.policy_loss_grad(x, t, None, torch.ones(2, device=x.device))
    assert loss.item() == 0 and kl.item() == 0 and not lps.any() and not dx.any()
    ids = torch.zeros(2, 5, 3, dtype=torch.int64, device=x.device)
    loss, dx = ops.distill_loss_grad(x, ids, ids.float(), torch.zeros_like(t, dtype=torch.bool))
    assert loss.item() == 0 and not dx.any()
    loss, rewards, dx = ops.preference_loss_grad(x, t)
    assert abs(loss.item() - math.log(2)) <= U and not rewards.any() and not dx.any()
    # no rows at all
    x0, t0 = x[:, :0], t[:, :0]
    assert ops.token_logprobs(x0, t0).shape == (2, 0)
    assert ops.policy_loss_grad(x0, t0, None, torch.ones(2, device=x.device))[0].item() == 0
    assert ops.distill_loss_grad(x0, ids[:, :0], ids[:, :0].float())[0].item() == 0
    assert abs(ops.preference_loss_grad(x0, t0)[0].item() - math.log(2)) <= U
    xr = x0.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.token_logprobs(xr, t0).sum(), xr)
    assert g.shape == x0.shape


def test_out_of_range_index_is_an_error(cuda_device):
    for bad in (400, -1, 2 ** 40):
        x, t, _ = make(cuda_device, 2, 5, 400, "bf16", ignore=0)
        t[0, 1] = bad
        lp = ops.token_logprobs(x, t)
        assert _native.device_error() == 0x106
        assert lp[0, 1].isnan() and torch.isfinite(lp).sum() == 9
        loss, _, dx = ops.preference_loss_grad(x, t)
        assert _native.device_error() == 0x106 and loss.isnan() and dx[0].isnan().all()
        loss, _, _, dx = ops.policy_loss_grad(x, t, None, torch.ones(2, device=x.device))
        assert _native.device_error() == 0x106 and loss.isnan() and dx[0, 1].isnan().all()
        assert torch.isfinite(dx[0, 0].float()).all()
        ids = torch.zeros(2, 5, 3, dtype=torch.int64, device=x.device)
        ids[0, 1, 2] = bad
        loss, dx = ops.distill_loss_grad(x, ids, torch.ones(2, 5, 3, device=x.device))
        assert _native.device_error() == 0x106 and loss.isnan() and dx[0, 1].isnan().all()
        assert torch.isfinite(dx[0, 0].float()).all()


def test_out_argument(cuda_device):
    for dtype, V in (("bf16", 32000), ("bf16", 5003), ("fp32", 50257), ("bf16", 300001)):
        x, t, _ = make(cuda_device, 2, 9, V, dtype)
        adv = torch.ones(2, device=x.device)
        tl, ids = torch.topk(x.float(), 8, -1)
        for f in (lambda v, o: ops.policy_loss_grad(v, t, None, adv, out=o),
                  lambda v, o: ops.preference_loss_grad(v, t, out=o),
                  lambda v, o: ops.distill_loss_grad(v, ids, tl, t != IGN, out=o)):
            want = f(x, None)
            y = x.clone()
            version = y._version
            got = f(y, y)
            assert got[-1] is y and y._version > version
            for a, b in zip(want, got):
                assert torch.equal(a, b)
            guard = torch.full((2, 9, V + 5), 7.0, dtype=x.dtype, device=x.device)
            f(x, guard[..., 3:3 + V])
            assert torch.equal(guard[..., 3:3 + V], want[-1])
            assert (guard[..., :3] == 7).all() and (guard[..., 3 + V:] == 7).all()
    x, t, _ = make(cuda_device, 2, 9, 64, "bf16")
    big = torch.empty(2, 10, 64, dtype=x.dtype, device=x.device)
    for out in (x[:, :, :32], x.float(), big[:1, :9].expand(2, 9, 64),
                torch.empty(2, 64, 9, dtype=x.dtype, device=x.device).transpose(1, 2),
                x.clone().requires_grad_(True)):
        with pytest.raises(ValueError):
            ops.preference_loss_grad(x, t, out=out)
    big[:, :9] = x
    with pytest.raises(ValueError, match="shares"):
        ops.preference_loss_grad(big[:, :9], t, out=big[:, 1:])


def test_refusals(cuda_device):
    x, t, _ = make(cuda_device, 2, 4, 50, "bf16")
    f = torch.zeros(2, 4, device=x.device)
    adv = torch.zeros(2, device=x.device)
    ids = torch.zeros(2, 4, 3, dtype=torch.int64, device=x.device)
    tl = ids.float()
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), t)
    with pytest.raises(TypeError):
        ops.token_logprobs(x, t.int())
    with pytest.raises(ValueError):
        ops.token_logprobs(x, t[:, :3])
    with pytest.raises(ValueError):
        ops.token_logprobs(x[0, 0], t[0, 0])
    with pytest.raises(ValueError):
        ops.token_logprobs(x[..., :0], t)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, t.cpu())
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        with pytest.raises(_native.LemaError, match="temperature"):
            ops.token_logprobs(x, t, temperature=tau)
    with pytest.raises(ValueError):
        ops.preference_loss(x[:1], t[:1])
    with pytest.raises(ValueError):
        ops.preference_loss(x.view(8, 50), t.view(8))
    with pytest.raises(ValueError, match="detach"):
        ops.preference_loss(x, t, f.clone().requires_grad_(True))
    for kw in ({"beta": 0.0}, {"beta": float("nan")}, {"label_smoothing": 0.5},
               {"label_smoothing": -0.1}):
        with pytest.raises(_native.LemaError):
            ops.preference_loss(x, t, **kw)
    with pytest.raises(ValueError):
        ops.policy_loss(x, t, f, torch.zeros(4, device=x.device))
    with pytest.raises(ValueError):
        ops.policy_loss(x, t, f, adv.double())
    with pytest.raises(ValueError):
        ops.policy_loss(x, t, f, adv, reduction="mean")
    for kw in ({"clip": (-0.1, 0.2)}, {"clip": (0.2, float("inf"))}, {"clip": (1.5, 0.2)},
               {"kl_coef": -1.0}):
        with pytest.raises(_native.LemaError):
            ops.policy_loss(x, t, f, adv, **kw)
    with pytest.raises(TypeError):
        ops.distill_loss(x, ids.float(), tl)
    with pytest.raises(ValueError):
        ops.distill_loss(x, ids, tl[..., :2])
    with pytest.raises(TypeError):
        ops.distill_loss(x, ids, tl, torch.ones(2, 4, device=x.device))
    with pytest.raises(_native.LemaError):
        ops.distill_loss(x, ids[..., :0], tl[..., :0])
    with pytest.raises(_native.LemaError):
        big = torch.zeros(2, 4, 1025, device=x.device)
        ops.distill_loss(x, big.long(), big)


def test_autograd_use(cuda_device):
    """Twice through a retained graph, a modified input, no second derivative, an
    expanded upstream gradient, a loss added to others."""
    x, t, _ = make(cuda_device, 2, 6, 700, "fp32")
    xr = x.clone().requires_grad_(True)
    loss, _ = ops.preference_loss(xr, t)
    (a,) = torch.autograd.grad(loss, xr, retain_graph=True)
    (b,) = torch.autograd.grad(loss, xr)
    assert torch.equal(a, b)
    lp = ops.token_logprobs(xr, t)
    (s,) = torch.autograd.grad(lp.sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(s.sum(), xr)
    y = (x * 1.0).requires_grad_(True)
    z = y * 1.0
    lp = ops.token_logprobs(z, t)
    z.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        lp.sum().backward()
    h = x.clone().requires_grad_(True)
    w = torch.randn(700, 700, device=x.device) * 0.02
    logits = (h @ w).bfloat16()
    total = ops.policy_loss(logits, t, None, torch.ones(2, device=x.device))[0] \
        - ops.token_logprobs(logits, t).mean()
    total.backward()
    assert torch.isfinite(h.grad).all() and h.grad.abs().sum() > 0


def test_same_bits_every_time(cuda_device):
    x, t, _ = make(cuda_device, 4, 150, 8200, "bf16")
    tl, ids = torch.topk(x.float(), 32, -1)
    ids[..., 7] = ids[..., 3]
    adv = torch.randn(4, device=x.device)
    for f in (lambda: ops.preference_loss_grad(x, t), lambda: ops.distill_loss_grad(x, ids, tl),
              lambda: ops.policy_loss_grad(x, t, None, adv, reduction="sequence")):
        first = f()
        for _ in range(3):
            for a, b in zip(first, f()):
                assert torch.equal(a, b)


def test_streams_and_graphs(cuda_device):
    """On another stream than the default; captured, replayed on new inputs; two graphs
    captured one after the other and replayed at once (each has its own workspace)."""
    dev = cuda_device
    data = [make(dev, 4, 40, 5000, "bf16", seed=s) for s in range(4)]
    adv = torch.randn(4, device=dev)
    want = [(ops.preference_loss_grad(x, t), ops.policy_loss_grad(x, t, None, adv))
            for x, t, _ in data]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = ops.preference_loss_grad(data[1][0], data[1][1])
    side.synchronize()
    for a, b in zip(want[1][0], got):
        assert torch.equal(a, b)
    graphs = []
    for i in range(2):
        x, t = data[i][0].clone(), data[i][1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = (ops.preference_loss_grad(x, t), ops.policy_loss_grad(x, t, None, adv))
        graphs.append((g, x, t, outs))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for round_ in (0, 2):
        for (g, x, t, _), (nx, nt, _) in zip(graphs, data[round_:round_ + 2]):
            x.copy_(nx)
            t.copy_(nt)
        torch.cuda.synchronize()
        for _ in range(5):
            for s, (g, *_) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (_, _, _, outs), w in zip(graphs, want[round_:round_ + 2]):
            for a, b in zip([v for o in outs for v in o], [v for o in w for v in o]):
                assert torch.equal(a, b)


def test_backward_in_a_graph(cuda_device):
    """Forward and backward of the autograd form captured together."""
    x, t, _ = make(cuda_device, 2, 30, 3000, "bf16")
    want = ops.preference_loss_grad(x, t)
    xr = x.clone().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, _ = ops.preference_loss(xr, t)
        (dx,) = torch.autograd.grad(loss, xr)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss.detach(), want[0]) and torch.equal(dx, want[2])


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 logits: the last rows against their own small call."""
    T, V = 68000, 32000
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=cuda_device)
    t = torch.full((T,), IGN, device=cuda_device)
    tail, tt, _ = make(cuda_device, 1, 6, V, "bf16", ignore=0)
    x[-6:] = tail[0]
    t[-6:] = tt[0]
    adv = torch.ones(T, device=cuda_device)
    # a small call spreads a row over other threads: its sums may round otherwise, so both are
    # held to fp64
    want, q = ref_logps(tail, tt)
    loss, lps, _, dx = ops.policy_loss_grad(x, t, None, adv, out=x)
    assert abs(loss.item() + 1.0) <= 2 * U
    check_logps(lps[None, -6:], want, V)
    k = torch.full((1, 6), -1.0 / 6, dtype=torch.float64, device=x.device)
    check_dx(dx[None, -6:], tail, q, k, onehot(tt, V))
    assert not lps[:-6].any() and not dx[:-6].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S,V", [(8, 900, 9001), (3, 4000, 257), (2, 250, 33001)])
def test_many_rows(cuda_device, B, S, V, dtype):
    """More rows than CTAs times the rows in flight, long runs of ignored ones among them."""
    x, t, g = make(cuda_device, B, S, V, dtype)
    t[0, S // 4:S // 2] = IGN
    t[-1, :S // 3] = IGN
    adv = torch.randn(B, device=x.device, generator=g)
    n = int((t != IGN).sum())
    tl, ids = torch.topk(x.float(), 5, -1)
    loss, lps, _, dx = ops.policy_loss_grad(x, t, None, adv)
    lossd, dxd = ops.distill_loss_grad(x, ids, tl, t != IGN)
    want = wantd = 0.0
    for b in range(B):
        lp, q = ref_logps(x[b:b + 1], t[b:b + 1])
        check_logps(lps[b:b + 1], lp, V)
        k = torch.where(t[b:b + 1] == IGN, 0.0, -adv[b].double() / n)
        check_dx(dx[b:b + 1], x[b:b + 1], q, k, onehot(t[b:b + 1], V))
        want -= (adv[b].double() * (t[b] != IGN).sum() / n).item()
        m = t[b:b + 1] != IGN
        part, kd, mass, _ = ref_distill(x[b:b + 1], ids[b:b + 1], tl[b:b + 1], m, 1.0)
        share = int(m.sum()) / n
        wantd += part.item() * share
        check_dx(dxd[b:b + 1], x[b:b + 1], q, kd * share, mass)
    assert abs(loss.item() - want) <= 4 * U * adv.abs().mean().item() + 2 * U * abs(want)
    assert abs(lossd.item() - wantd) <= rel_s(V) + 60 * U + 2 * U * abs(wantd)


@pytest.mark.parametrize("B,S,V", [(600, 20, 300), (600, 15, 8500), (30, 30, 9001), (2, 3, 40000)])
def test_many_sequences(cuda_device, B, S, V):
    """Means over each sequence's tokens, whose counts differ, at row counts listed by one
    CTA, by several and by every CTA for itself; sequences without a counted token."""
    x, t, g = make(cuda_device, B, S, V, "bf16", ignore=0.4)
    t[B // 2] = IGN
    adv = torch.randn(B, S, device=x.device, generator=g)
    loss, lps, _, dx = ops.policy_loss_grad(x, t, None, adv, reduction="sequence")
    n = (t != IGN).sum(1, keepdim=True)
    w = torch.where(t == IGN, 0.0, 1.0 / (B * n.clamp(min=1).double()))
    want = -(w * adv.double()).sum().item()
    assert abs(loss.item() - want) <= 2 * U * abs(want) + 1e-12
    for b in range(0, B, 50):
        e = min(B, b + 50)
        lp, q = ref_logps(x[b:e], t[b:e])
        check_logps(lps[b:e], lp, V)
        check_dx(dx[b:e], x[b:e], q, -w[b:e] * adv[b:e].double(), onehot(t[b:e], V))
    again = ops.policy_loss_grad(x, t, None, adv, reduction="sequence")
    assert torch.equal(again[0], loss) and torch.equal(again[3], dx)


@pytest.mark.parametrize("V", [9001, 40000, 300001])
def test_long_rows_in_graphs(cuda_device, V):
    """Captured and replayed on other inputs: rows held by one CTA, by clusters, and swept."""
    dev = cuda_device
    data = [make(dev, 4, 9, V, "bf16", seed=s) for s in range(2)]
    tl = [torch.topk(x.float(), 40, -1) for x, _, _ in data]
    adv = torch.randn(4, device=dev)

    def all_of(x, t, v, i):
        return (*ops.policy_loss_grad(x, t, None, adv, reduction="sequence"),
                *ops.preference_loss_grad(x, t), *ops.distill_loss_grad(x, i, v, t != IGN))
    want = [all_of(x, t, v, i) for (x, t, _), (v, i) in zip(data, tl)]
    bufs = [data[0][0].clone(), data[0][1].clone(), tl[0][0].clone(), tl[0][1].clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of(*bufs)
    for k in (1, 0, 1):
        for b, src in zip(bufs, (data[k][0], data[k][1], tl[k][0], tl[k][1])):
            b.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, want[k]):
            assert torch.equal(a, w)


def test_most_teacher_entries_on_long_rows(cuda_device):
    """Entries that leave little room beside rows that fill a CTA and a cluster; each index
    twice."""
    for S, V, K in ((70, 32000, 512), (310, 32000, 512), (310, 32000, 300), (310, 20000, 220),
                    (70, 70000, 512), (5, 100000, 512), (3, 250001, 512), (310, 9001, 512)):
        x, _, _ = make(cuda_device, 1, S, V, "bf16")
        val, ids = torch.topk(x.float(), K, -1)
        ids, val = torch.cat([ids, ids.flip(-1)], -1), torch.cat([val, val.flip(-1) - 1], -1)
        loss, dx = ops.distill_loss_grad(x, ids, val)
        want, k, mass, q = ref_distill(x, ids, val, None, 1.0)
        # A weight is off by 7 u (its exponent spans less than 7), 2 u (ex2), 37 u (the sum of
        # 32 a lane and of the lanes) and 2 u (the division and the sum of two): 48 u. The terms
        # p (log p - log q) take that times |log p - log q| < 2 or so, and 9 u of log p.
        assert abs(loss.item() - want.item()) <= rel_s(V) + 110 * U + 2 * U * abs(want.item())
        check_dx(dx, x, q, k, mass, mass_err=48 * U)


@pytest.mark.parametrize("V", [5000, 9001, 70000])
def test_far_rows(cuda_device, V):
    """Logits and temperatures whose exponents leave the range of one reference, in rows kept
    as exponentials, held by one CTA and shared by several."""
    g = torch.Generator(device=cuda_device).manual_seed(V)
    for dtype in (torch.bfloat16, torch.float32):
        for lift, tau in ((0.0, 1e-3), (3e4, 1.0), (-3e4, 1.0), (30.0, 100.0), (1e30, 1.0)):
            x = torch.randn(1, 6, V, device=cuda_device, generator=g)
            # steps that the lifted values keep, the top of them a few apart
            x = (x.round() * (max(lift * lift, 1.0) ** 0.5 / 128 if lift else 1.0) + lift).to(dtype)
            t = torch.stack([x[0].float().argmax(-1), x[0].float().argmin(-1)], -1)[None]
            t = torch.where(torch.arange(6, device=x.device) % 2 == 0, t[..., 0], t[..., 1])
            adv = torch.ones(1, 6, device=x.device)
            loss, lps, _, dx = ops.policy_loss_grad(x, t, None, adv, temperature=tau)
            lp, q = ref_logps(x, t, tau)
            # the difference of two values, times 1 / tau, is rounded thrice
            tol = rel_s(V) + 12 * U + 4 * U * lp.abs()
            assert ((lps.double() - lp).abs() <= tol).all()
            # k = -1/6/tau (mass - q); the bound on q counts exponents up to 150
            check_dx(dx, x, q, torch.full((1, 6), -1 / 6 / tau, dtype=torch.float64,
                                          device=x.device), onehot(t, V), tau)


@pytest.mark.parametrize("V", [8201, 13001, 18440, 33000, 70001, 80000, 96777, 136001, 176008,
                               208003, 258048])
def test_row_lengths(cuda_device, V):
    """Rows that one CTA of either size holds, and that two to eight share."""
    dtype = "bf16"
    for B, S in ((2, 2), (2, 75)):
        x, t, g = make(cuda_device, B, S, V, dtype)
        adv = torch.randn(B, S, device=x.device, generator=g)
        loss, lps, _, dx = ops.policy_loss_grad(x, t, None, adv)
        lp, q = ref_logps(x, t)
        check_logps(lps, lp, V)
        n = max(1, int((t != IGN).sum()))
        check_dx(dx, x, q, torch.where(t == IGN, 0.0, -adv.double() / n), onehot(t, V))
        val, ids = torch.topk(x.float(), 7, -1)
        _, dx = ops.distill_loss_grad(x, ids, val, t != IGN)
        _, k, mass, q = ref_distill(x, ids, val, t != IGN, 1.0)
        # the weights' own errors: 7 u of their exponents, 2 u of ex2, 7 u of their sum, 2 u
        check_dx(dx, x, q, k, mass, mass_err=18 * U)
        del x, q, mass, dx


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [5, 37, 300, 1999, 8000, 9001, 33000, 300001])
def test_gradient_rows_at_other_phases(cuda_device, V, dtype):
    """Gradient rows that start at every place within 16 bytes, whatever their logits' place; what
    lies between them stays."""
    x, t, g = make(cuda_device, 2, 9, V, dtype, ignore=0.2)
    adv = torch.randn(2, 9, device=x.device, generator=g)
    val, ids = torch.topk(x.float(), min(V, 5), -1)
    w = torch.where(t == IGN, 0.0, adv).contiguous()
    lead = x.requires_grad_(True)
    want = [ops.policy_loss_grad(x.detach(), t, None, adv)[3],
            ops.distill_loss_grad(x.detach(), ids, val, t != IGN)[1],
            ops.preference_loss_grad(x.detach(), t)[2]]
    lp = torch.autograd.grad(ops.token_logprobs(lead, t), lead, w)[0]
    x = x.detach()
    for gap in range(1, 9 if dtype == "bf16" else 5):
        room = torch.full((2, 9, V + 16), 7.0, dtype=x.dtype, device=x.device)
        out = room[..., gap:gap + V]
        shut = (room[..., :gap], room[..., gap + V:])
        for k, f in enumerate((lambda: ops.policy_loss_grad(x, t, None, adv, out=out),
                               lambda: ops.distill_loss_grad(x, ids, val, t != IGN, out=out),
                               lambda: ops.preference_loss_grad(x, t, out=out))):
            f()
            assert torch.equal(out, want[k])
            assert all((s == 7.0).all() for s in shut)
        # the same from logits at another place
        apart = torch.empty(2, 9, V + 16, dtype=x.dtype, device=x.device)[..., gap:gap + V]
        apart.copy_(x).requires_grad_(True)
        got = torch.autograd.grad(ops.token_logprobs(apart, t), apart, w)[0]
        # edges differ, and with them the order of a row's sum
        tol = half_step(got.dtype) * 2.1 * lp.double().abs() + rel_s(V) * w[..., None].abs()
        assert ((got.double() - lp.double()).abs() <= tol).all()


@pytest.mark.parametrize("V", [130, 8500])
def test_many_rows_in_graphs(cuda_device, V):
    """Rows that a cluster lists, captured: what is counted at replay is what the targets say
    then. Two streams replay two graphs at once."""
    dev = cuda_device
    data = [make(dev, 45, 200, V, "bf16", seed=s, ignore=0.2 + 0.3 * s) for s in range(2)]
    adv = torch.randn(45, device=dev)

    def both(x, t):
        return (*ops.policy_loss_grad(x, t, None, adv, reduction="sequence"),
                *ops.policy_loss_grad(x, t, None, adv))
    want = [both(x, t) for x, t, _ in data]
    graphs = []
    for x, t, _ in data:
        bufs = [x.clone(), t.clone()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = both(*bufs)
        graphs.append((g, bufs, got))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for swap in (1, 0):
        for k, (_, bufs, _) in enumerate(graphs):
            for b, src in zip(bufs, data[k ^ swap]):
                b.copy_(src)
        torch.cuda.synchronize()
        for s, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for k, (_, _, got) in enumerate(graphs):
            for a, w in zip(got, want[k ^ swap]):
                assert torch.equal(a, w)


@pytest.mark.parametrize("V,K,dtype", [(7, 300, "bf16"), (300, 1024, "fp32"), (520, 40, "bf16"),
                                       (2055, 244, "bf16"), (1802, 64, "fp32"), (8190, 700, "bf16")])
def test_repeated_entries_of_short_rows(cuda_device, V, K, dtype):
    """Indices drawn with repetition, and all alike, in rows that a warp or 128 threads hold."""
    x, _, g = make(cuda_device, 2, 21, V, dtype)
    val = torch.randn(2, 21, K, device=x.device, generator=g)
    ids = torch.randint(0, V, (2, 21, K), device=x.device, generator=g)
    ids[0, 0] = V - 1
    ids[1, 3] = V - 1 - (torch.arange(K, device=x.device) % 2)
    for kind in (torch.int64, torch.int32):
        loss, dx = ops.distill_loss_grad(x, ids.to(kind), val)
        want, k, mass, q = ref_distill(x, ids, val, None, 1.0)
        # a weight: exponents below 16 (16 u), ex2 and expf 4 u, a sum of 32 a lane and the lanes
        # 37 u; repeated ones are added in fp32, K / 4 in a row: K / 4 u
        err = (57 + K / 4) * U
        check_dx(dx, x, q, k, mass, mass_err=err)
        assert abs(loss.item() - want.item()) <= rel_s(V) + 8 * err + 2 * U * abs(want.item())


def _straddling_rows(dev, dtype, V, seed):
    """Rows around |x log2 e| = 2048 (|x| = 1419.565), where the statistics of a preference row
    change their reference, on both sides of zero; rows short of it and wholly beyond."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = []
    for sign in (1.0, -1.0):
        for mean, std in ((1300.0, 2.0), (1412.0, 2.0), (1416.0, 4.0), (1418.75, 0.3),
                          (1419.5, 0.1), (1420.5, 0.3), (1427.0, 2.0), (1500.0, 2.0),
                          (3e4, 2.0)):
            rows.append(sign * mean + std * torch.randn(V, device=dev, generator=g))
        # two values, the higher one rare: at the front, at the end, anywhere
        low, high = sorted((sign * 1416.0, sign * 1424.0)) if dtype is torch.bfloat16 else \
            sorted((sign * 1419.25, sign * 1419.75))
        for at in (0, V - 1, V // 3):
            row = torch.full((V,), low, device=dev)
            row[at] = high
            rows.append(row)
        ramp = torch.linspace(low - 8, high + 8, V, device=dev)   # every step a new maximum
        rows += [ramp, ramp.flip(0)]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [300, 2000, 7001, 16001, 40000])
def test_preference_rows_across_the_far_border(cuda_device, V, dtype):
    """Maxima on both sides of the border between the threads of a row and between their
    sweeps (rows held by a warp, by 128 threads in one and in two sweeps, by 512). Sequences
    of one token, so that each reward is a log-probability. A partial sum crosses the border
    once within its thread and once when the threads meet: each multiplies by a power of two
    whose exponent e is rounded to u |e| (weighted by 2^-|e|, less than u) and taken by
    ex2.approx (4 u): 10 u beside the bound of any row."""
    x = _straddling_rows(cuda_device, DT[dtype], V, V)
    n = x.shape[0]
    g = torch.Generator(device=cuda_device).manual_seed(3)
    t = torch.where(torch.arange(n, device=x.device) % 2 == 0, x.float().argmax(-1),
                    torch.randint(0, V, (n,), device=x.device, generator=g))[:, None]
    x = torch.cat([x, x.flip(0)])[:, None]          # each row chosen once and rejected once
    t = torch.cat([t, t.flip(0)])
    P = n
    lp, q = ref_logps(x, t)
    ref = (lp + 0.3 * torch.randn(lp.shape, device=x.device, generator=g,
                                  dtype=torch.float64)).float()
    lp_err = rel_s(V) + 10 * U
    a_max = min((x.double().amax(-1) - x.double().amin(-1)).max().item() * 1.4427, 150.0)
    mass = onehot(t, V)
    for r, e in ((None, 0.0), (ref, 0.1)):
        loss, rewards, dx = ops.preference_loss_grad(x, t, r, beta=1.0, label_smoothing=e)
        want, R, k, _ = ref_preference(x, t, r, 1.0, e)
        assert ((rewards.double() - R).abs() <= lp_err + U * R.abs()).all(), \
            (rewards.double() - R).abs().max().item()
        assert abs(loss.item() - want.item()) <= 2 * lp_err + 2 * U * abs(want.item())
        # dL/dh moves by at most a quarter of h's error
        slack = 2 * lp_err / 4 / P
        wantx = k[..., None] * (mass - q)
        tol = (half_step(x.dtype) + 8 * U) * wantx.abs() \
            + k.abs()[..., None] * (q * (lp_err + (4 + 2.1 * a_max) * U) + 2 * U * mass) \
            + slack * (mass - q).abs() + 1e-37
        assert ((dx.double() - wantx).abs() <= tol).all()
        xr = x.clone().requires_grad_(True)
        l2, rw2 = ops.preference_loss(xr, t, r, beta=1.0, label_smoothing=e)
        assert torch.equal(l2.detach(), loss) and torch.equal(rw2, rewards)
        assert torch.equal(torch.autograd.grad(l2, xr)[0], dx)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [3, 400, 9001])
def test_gradient_of_an_out_of_range_target(cuda_device, V, dtype):
    """Under autograd, too, a bad target's outputs are NaN: its log-probability, statistics and
    gradient row (whatever its upstream gradient), and no other row's."""
    for bad in (V, -1, 2 ** 40):
        x, t, _ = make(cuda_device, 2, 5, V, dtype, ignore=0)
        t[0, 1] = bad
        t[1, 4] = IGN
        hit = torch.zeros(2, 5, dtype=torch.bool, device=x.device)
        hit[0, 1] = True
        adv = torch.ones(2, 5, device=x.device)
        for f in (lambda v: ops.token_logprobs(v, t).nansum(),
                  lambda v: ops.token_logprobs(v, t).sum(),
                  lambda v: ops.policy_loss(v, t, None, adv)[0]):
            xr = x.clone().requires_grad_(True)
            loss = f(xr)
            assert _native.device_error() == 0x106
            (dx,) = torch.autograd.grad(loss, xr)
            assert dx[hit].isnan().all() and torch.isfinite(dx[~hit]).all()
            assert (dx[1, 4] == 0).all()
        xr = x.clone().requires_grad_(True)
        (dx,) = torch.autograd.grad(ops.token_logprobs(xr, t), xr, torch.zeros_like(adv))
        assert _native.device_error() == 0x106
        assert dx[hit].isnan().all() and (dx[~hit] == 0).all()
        stats = torch.zeros(2, 5, 2, device=x.device)
        lp = torch.zeros(2, 5, device=x.device)
        _native.call("lema_token_logprobs", x.data_ptr(), int(dtype == "fp32"), 2, 5, 5 * V, V, V,
                     t.data_ptr(), IGN, 1.0, lp.data_ptr(), stats.data_ptr(),
                     torch.cuda.current_stream().cuda_stream)
        assert _native.device_error() == 0x106
        assert stats[..., 1][hit].isnan().all() and torch.isfinite(stats[~hit]).all()


# rows held by a warp, by 128 threads, by a CTA and by a cluster, and swept
POLICY_LENGTHS = [300, 5000, 9001, 70000, 300001]


def _even_rows(dev, B, S, V, dtype):
    """Rows of one value. Their sum is V (exact below 2^24) and each log-probability -log V, so
    that what the loss makes of it can be held to fp64 without the rows' own rounding."""
    x = torch.zeros(B, S, V, dtype=DT[dtype], device=dev)
    t = torch.randint(0, V, (B, S), device=dev, generator=torch.Generator(dev).manual_seed(V))
    return x, t, torch.full((B, S), -math.log(V), dtype=torch.float64, device=dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", POLICY_LENGTHS)
def test_kl_slope_of_a_policy_near_its_reference(cuda_device, V, dtype):
    """Advantages of 0 and |ref - lp| from 1e-5 to 0.2: the row is -kl_coef (e^d - 1) w alone.
    Relative bound: for fp32 rows d and e^d - 1 round once each (2 u and 2 u), kl_coef, w and
    three products 5 u, 1 / s and two products behind it 4 u: 16 u in all with the stored
    value's; for bf16 e^d - 1 is 8e-6 off (the remainder d^3 / 24 below 1/32, 2.4e-7 of
    e^d above), 1e-5 with the rest."""
    x, t, lp = _even_rows(cuda_device, 4, 12, V, dtype)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    size = 10.0 ** (-5 + 4.3 * torch.rand(4, 12, device=x.device, generator=g))
    sign = torch.where(torch.rand(4, 12, device=x.device, generator=g) < 0.5, -1.0, 1.0)
    ref = (lp + (size * sign).double()).float()
    d = ref.double() - lp
    adv = torch.zeros(4, device=x.device)
    k = -0.3 * torch.expm1(d) / 48
    mass = onehot(t, V)
    want = k[..., None] * (mass - 1.0 / V)
    rel = half_step(x.dtype) + 1e-5 if dtype == "bf16" else 16 * U
    old = (lp + 0.05).float()
    for o in (None, old):
        dx = ops.policy_loss_grad(x, t, o, adv, ref, kl_coef=0.3)[3]
        assert ((dx.double() - want).abs() <= rel * want.abs()).all(), \
            ((dx.double() - want).abs() / want.abs()).max().item()
        xr = x.clone().requires_grad_(True)
        (dx,) = torch.autograd.grad(ops.policy_loss(xr, t, o, adv, ref, kl_coef=0.3)[0], xr)
        assert ((dx.double() - want).abs() <= rel * want.abs()).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", POLICY_LENGTHS)
def test_ratios_next_to_the_clip_ends(cuda_device, V, dtype):
    """Ratios a few last places of an old log-probability on either side of the clip range's
    ends: both forms clip those that the fp64 formula clips, and no others."""
    x, t, lp = _even_rows(cuda_device, 2, 42, V, dtype)
    up = torch.arange(42, device=x.device)
    for tau in (1.0, 0.7):
        for clip in ((0.2, 0.3), (0.05, 0.28)):
            edge = torch.tensor([math.log(1 - clip[0]), math.log(1 + clip[1])], device=x.device,
                                dtype=torch.float64)[:, None]
            # 21 steps of fp32 below and 21 above
            step = 2.0 ** (math.floor(math.log2(math.log(V))) - 23)
            old = ((lp - edge).float().double() + (up - 21) * step).float()
            r = lp - old.double() - edge   # above 0: past the upper end, inside the lower
            assert r.abs().min() > 1e-11              # log_sum is good to 1e-13
            adv = torch.where(torch.arange(2, device=x.device) == 0, -1.0, 1.0)   # per sequence
            gone = torch.stack([r[0] < 0, r[1] > 0])
            dx = ops.policy_loss_grad(x, t, old, adv, clip=clip, temperature=tau)[3]
            assert torch.equal((dx == 0).all(-1), gone)
            xr = x.clone().requires_grad_(True)
            (dx,) = torch.autograd.grad(
                ops.policy_loss(xr, t, old, adv, clip=clip, temperature=tau)[0], xr)
            assert torch.equal((dx == 0).all(-1), gone)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", POLICY_LENGTHS)
def test_both_forms_of_the_policy_gradient(cuda_device, V, dtype):
    """One call and autograd on ordinary rows, ratios anywhere and the reference near: the same
    row statistics and the same fp64 differences, so what is between them is the rounding of the
    coefficient (1e-5 for bf16 rows, 16 u) and of each stored value."""
    x, t, g = make(cuda_device, 2, 14, V, dtype)
    lp, _ = ref_logps(x, t, 0.9)
    shape = lp.shape
    noise = torch.randn(shape, device=x.device, generator=g, dtype=torch.float64)
    old = (lp - 0.3 * noise).float()
    ref = (lp + 3e-4 * noise.flip(0)).float()
    adv = torch.randn(shape, device=x.device, generator=g)
    adv[:, ::2] = 0.0
    coef = 1e-5 if dtype == "bf16" else 16 * U
    for kl in (0.0, 0.5):
        kw = dict(kl_coef=kl, temperature=0.9, reduction="sequence")
        dx = ops.policy_loss_grad(x, t, old, adv, ref, **kw)[3]
        xr = x.clone().requires_grad_(True)
        (gx,) = torch.autograd.grad(ops.policy_loss(xr, t, old, adv, ref, **kw)[0], xr)
        assert torch.equal((dx == 0).all(-1), (gx == 0).all(-1))
        a, b = dx.double(), gx.double()
        # the target's own value is a difference of k and k q: its bound goes by the row's largest
        top = torch.maximum(a.abs(), b.abs()).amax(-1, keepdim=True)
        tol = (2 * half_step(x.dtype) + 2 * coef) * torch.maximum(a.abs(), b.abs()) \
            + 8 * U * onehot(t, V) * top + 1e-37
        assert ((a - b).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [130, 2000, 9001, 40000])
def test_preference_of_infinities_and_lowest_values(cuda_device, V, dtype):
    """Masked vocabularies through the preference loss's own statistics, each row a sequence of
    its own beside an ordinary one, chosen and rejected."""
    low = torch.finfo(DT[dtype]).min
    x, _, _ = make(cuda_device, 1, 8, V, dtype, ignore=0)
    x = x[0][:, None]
    x[0, 0, 10:] = float("-inf")
    x[1] = low
    x[2] = low
    x[2, 0, 3] = 0.0
    x[3, 0, 3] = float("-inf")           # the target itself masked
    x[4] = float("-inf")
    x[5, 0, 7] = float("nan")
    x[6, 0, 5] = float("inf")
    plain, _, _ = make(cuda_device, 8, 1, V, dtype, seed=5, ignore=0)
    t = torch.full((16, 1), 3, device=x.device)
    for both in (torch.cat([x, plain]), torch.cat([plain, x])):
        z = both.double()
        lsm = torch.log_softmax(z - z.amax(-1, keepdim=True), -1)
        want = lsm[..., 3].sum(1)
        _, rewards, dx = ops.preference_loss_grad(both, t, beta=1.0)
        got = rewards.double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        ok = torch.isfinite(want)
        assert ((got - want).abs()[ok] <= (rel_s(V) + U * want.abs())[ok]).all()
        bad = want[:8].isnan() | want[8:].isnan()
        assert dx[torch.cat([bad, bad])].isnan().all()
        h = want[:8] - want[8:]
        k = torch.cat([-torch.sigmoid(-h), torch.sigmoid(-h)]) / 8
        for r in (~torch.cat([bad, bad])).nonzero().flatten().tolist():
            q = lsm[r, 0].exp()
            mass = torch.zeros_like(q)
            mass[3] = 1
            w = k[r] * (mass - q)
            tol = (half_step(x.dtype) + 8 * U) * w.abs() \
                + k[r].abs() * (q * (rel_s(V) + 300 * U) + 2 * U * mass) \
                + 2 * rel_s(V) / 8 * (mass - q).abs() + 1e-37
            assert ((dx[r, 0].double() - w).abs() <= tol).all(), r


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [130, 5000, 9001, 70000, 300001])
def test_terms_without_weight(cuda_device, V, dtype):
    """A target without probability (its logit -inf) where its infinite term has weight 0:
    a rejected token without smoothing, the KL with a coefficient of 0."""
    x, t, _ = make(cuda_device, 2, 3, V, dtype, ignore=0)
    x[1, 1, t[1, 1]] = float("-inf")
    loss, rewards, dx = ops.preference_loss_grad(x, t)
    assert loss.item() == 0.0 and rewards[1].item() == -math.inf and not dx.any()
    loss, _, _ = ops.preference_loss_grad(x, t, label_smoothing=0.1)
    assert loss.item() == math.inf
    old = ref = torch.full((2, 3), -2.0, device=x.device)
    adv = torch.ones(2, device=x.device)
    loss, lps, kl, dx = ops.policy_loss_grad(x, t, old, adv, ref)
    plain = ops.policy_loss_grad(x, t, old, adv)
    assert kl.item() == math.inf and torch.isfinite(loss) and torch.isfinite(dx).all()
    assert torch.equal(loss, plain[0]) and torch.equal(dx, plain[3]) and not dx[1, 1].any()
    loss, _, _, dx = ops.policy_loss_grad(x, t, old, adv, ref, kl_coef=0.1)
    assert loss.item() == math.inf and not torch.isfinite(dx[1, 1]).any()


def test_no_rows_of_any_shape(cuda_device):
    for lead in ((0,), (2, 0), (0, 3), (2, 2, 0), (0, 2, 3), (2, 0, 3)):
        x = torch.zeros(*lead, 50, device=cuda_device, dtype=torch.bfloat16)
        t = torch.zeros(lead, dtype=torch.int64, device=cuda_device)
        ids = torch.zeros(*lead, 3, dtype=torch.int64, device=cuda_device)
        assert ops.token_logprobs(x, t).shape == lead
        adv = torch.zeros(lead, device=cuda_device)
        for out in (None, x):
            loss, lps, kl, dx = ops.policy_loss_grad(x, t, None, adv, out=out)
            assert loss.item() == 0 and kl.item() == 0 and lps.shape == lead and dx.shape == x.shape
            loss, dx = ops.distill_loss_grad(x, ids, ids.float(), out=out)
            assert loss.item() == 0 and dx.shape == x.shape
        xr = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(ops.token_logprobs(xr, t).sum(), xr)
        assert g.shape == x.shape


def test_preference_without_counted_rows_in_a_graph(cuda_device):
    """Many pairs and no counted token, captured with what reads the loss behind it: no row of
    the gradient has anything to do, and the loss is still complete when it is read."""
    dev = cuda_device
    x = torch.zeros(6000, 40, 8, dtype=torch.bfloat16, device=dev)
    t = torch.full((6000, 40), IGN, device=dev)
    graph = torch.cuda.CUDAGraph()
    got = torch.zeros(20, device=dev)
    with torch.cuda.graph(graph):
        for i in range(20):
            loss, rewards, dx = ops.preference_loss_grad(x, t)
            got[i].copy_(loss)
            loss.fill_(7.0)
            rewards.fill_(7.0)
    for _ in range(5):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert ((got - math.log(2)).abs() <= U).all()
        assert loss.item() == 7.0 and (rewards == 7.0).all() and not dx.any()
