"""Tuning operators on the GPU against their formulas in 64 bits: layer norm, log-probabilities of sampled tokens, the
clipped policy loss, the preference loss, the global gradient norm and clipping.

Tolerances count roundings. u = 2^-24 is half a step of fp32, eps/2 half a step of the output's type. The longest chain of
fp32 additions in a sum is 32 terms in a thread plus 10 levels of a tree (see the kernels), so a sum of n terms of either
sign is off by at most 42 u sum|term|; the handful of further operations per element is rounded up to 64 u in all."""
import math

import pytest
import torch

import ldrs_amd  # noqa: F401
from ldrs_amd.hip import nn as hnn
from ldrs_amd.hip import ops
from ldrs_amd.hip.arena import ParamArena

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def half(t):
    return torch.finfo(t.dtype).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol elementwise, `got` rounded once from a value inside that band."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def strided(t, extra, shift=0):
    """The same matrix inside a wider buffer: row stride shape[1] + extra, starting `shift` elements in."""
    R, C = t.shape
    buf = torch.full((R * (C + extra) + shift + 8,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[shift:shift + R * (C + extra)].view(R, C + extra)[:, :C]
    v.copy_(t)
    return v


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------
def norm_ref(x, w, b, eps, dy=None):
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    out = dict(mu=mu[:, 0], r=r[:, 0], xh=xh, y=xh * w + b)
    if dy is not None:
        dy = dy.double()
        g = dy * w
        mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        out.update(dx=r * (g - mg - xh * mgx), dw=(dy * xh).sum(0), db=dy.sum(0))
        out["dx_tol"] = 128 * U * r * (g.abs() + g.abs().mean(-1, keepdim=True)
                                       + (xh.abs() + 1) * (g * xh).abs().mean(-1, keepdim=True))
        # 128 u also covers the additions over the rows: at most 41 in a lane (R <= 21000 in 512 workgroups), the
        # workgroup's groups (32) and the reduction over the workgroups (32 + 16)
        out["dw_tol"] = 128 * U * (dy.abs() * (xh.abs() + 1)).sum(0)
        out["db_tol"] = 128 * U * dy.abs().sum(0)
    return out


NORM_SIZES = [(1, 1), (3, 1), (1, 2), (5, 7), (2, 8), (33, 9), (64, 33), (7, 63), (9, 64), (4, 65), (130, 127), (3, 256),
              (5, 257), (3, 300), (65, 512), (6, 513), (4, 600), (10, 800), (37, 825), (300, 1024), (5, 1025), (2, 2047),
              (3, 2049), (2, 4096), (3, 4097), (2, 8191), (2, 8192), (2100, 40), (7, 1500), (9, 3000),
              (11, 8000), (40, 500), (700, 20), (20, 1500), (13, 825), (16, 825), (17, 825)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,C", NORM_SIZES)
def test_layer_norm(dev, R, C, dtype):
    g = gen(R * 10007 + C)
    x = (torch.randn(R, C, device=dev, generator=g) * 2 + torch.randn(R, 1, device=dev, generator=g)).to(dtype)
    dy = torch.randn(R, C, device=dev, generator=g).to(dtype)
    w, b = torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    ref = norm_ref(x, w, b, 1e-5, dy)
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, 1e-5)
    assert y.dtype == dtype and mean.shape == rstd.shape == (R,)
    close(mean, ref["mu"], 42 * U * x.double().abs().mean(-1), "mean")
    close(rstd, ref["r"], 64 * U * ref["r"], "rstd")
    ytol = 64 * U * (ref["xh"].abs() * w.abs() + w.abs() + b.abs())
    close(y, ref["y"], ytol + half(y) * (ref["y"].abs() + ytol), "y")
    dx, dw, db = ops.layer_norm_bwd(dy, x, w, mean, rstd)
    close(dx, ref["dx"], ref["dx_tol"] + half(dx) * (ref["dx"].abs() + ref["dx_tol"]), "dx")
    close(dw, ref["dw"], ref["dw_tol"], "dweight")
    close(db, ref["db"], ref["db_tol"], "dbias")
    again = ops.layer_norm_bwd(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again)), "two runs, two answers"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C,extra,shift", [(300, 4, 0), (257, 3, 1), (825, 0, 3), (64, 1, 5), (2049, 7, 1)])
def test_layer_norm_strides_in_place_and_optional_parts(dev, C, extra, shift, dtype):
    R, g = 21, gen(C)
    x0 = torch.randn(R, C, device=dev, generator=g).to(dtype)
    dy0 = torch.randn(R, C, device=dev, generator=g).to(dtype)
    w = torch.randn(C, device=dev, generator=g)
    y0, mean, rstd = ops.layer_norm_fwd(x0, w, None, 1e-5)
    d0 = ops.layer_norm_bwd(dy0, x0, w, mean, rstd)
    x, dy, y, dx = (strided(t, extra, shift) for t in (x0, dy0, x0, x0))
    assert ops.layer_norm_fwd(x, w, None, 1e-5, out=y)[0] is y and torch.equal(y, y0)
    got = ops.layer_norm_bwd(dy, x, w, mean, rstd, dx=dx)
    assert got[0] is dx and all(torch.equal(p, q) for p, q in zip(got, d0))
    for t in (y, dx):  # nothing beside the rows was written
        flat = t.as_strided((R * (C + extra) + 8,), (1,), t.storage_offset())
        pad = torch.cat([flat[r * (C + extra) + C:(r + 1) * (C + extra)] for r in range(R)] + [flat[R * (C + extra):]])
        assert pad.isnan().all()
    # in place: y over x, dx over dy, dx over x
    xi = strided(x0, extra, shift)
    assert torch.equal(ops.layer_norm_fwd(xi, w, None, 1e-5, out=xi)[0], y0)
    for over in (0, 1):
        di, xi = strided(dy0, extra, shift), strided(x0, extra, shift)
        assert torch.equal(ops.layer_norm_bwd(di, xi, w, mean, rstd, dx=(di, xi)[over])[0], d0[0])
    # parts alone, and accumulation into gradients that are there
    assert torch.equal(ops.layer_norm_bwd(dy0, x0, w, mean, rstd, params=False)[0], d0[0])
    only = ops.layer_norm_bwd(dy0, x0, w, mean, rstd, dx=False)
    assert only[0] is None and torch.equal(only[1], d0[1]) and torch.equal(only[2], d0[2])
    aw, ab = torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    want = (aw * 0.5 + d0[1], ab * 0.5 + d0[2])
    ops.layer_norm_bwd(dy0, x0, w, mean, rstd, dx=False, dweight=aw, dbias=ab, beta=0.5)
    for p, q in zip((aw, ab), want):
        close(p, q, 2 * U * (q.double().abs() + p.double().abs() + 1), "beta")
    # no parameters at all
    ref = norm_ref(x0, None, None, 0.0, dy0)
    y, mean, rstd = ops.layer_norm_fwd(x0, eps=0.0)
    ytol = 64 * U * (ref["xh"].abs() + 1)
    close(y, ref["y"], ytol + half(y) * (ref["y"].abs() + ytol), "y without parameters")
    dx, dw, db = ops.layer_norm_bwd(dy0, x0, None, mean, rstd)
    assert dw is None
    close(dx, ref["dx"], ref["dx_tol"] + half(dx) * (ref["dx"].abs() + ref["dx_tol"]), "dx without parameters")


# more rows than a launch has groups for (every group walks several, the forward pass past 8192 workgroups, the backward
# pass past what is resident), remainders of the grids, and matrices on both sides of the 128 MB that are streamed from on
LARGE_NORMS = [(300000, 24), (40000, 600), (9001, 1100), (9000, 2100), (8200, 4100), (45001, 825), (83001, 825)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,C", LARGE_NORMS)
def test_layer_norm_of_many_rows(dev, R, C, dtype):
    g = gen(R + C)
    x = (torch.randn(R, C, device=dev, generator=g) * 2 + torch.randn(R, 1, device=dev, generator=g)).to(dtype)
    dy = torch.randn(R, C, device=dev, generator=g).to(dtype)
    w, b = torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, 1e-5)
    dx, dw, db = ops.layer_norm_bwd(dy, x, w, mean, rstd)
    ref = norm_ref(x, w, b, 1e-5, dy)
    close(mean, ref["mu"], 42 * U * x.double().abs().mean(-1), "mean")
    close(rstd, ref["r"], 64 * U * ref["r"], "rstd")
    ytol = 64 * U * (ref["xh"].abs() * w.abs() + w.abs() + b.abs())
    close(y, ref["y"], ytol + half(y) * (ref["y"].abs() + ytol), "y")
    close(dx, ref["dx"], ref["dx_tol"] + half(dx) * (ref["dx"].abs() + ref["dx_tol"]), "dx")
    # a column's additions in fp32: at most 41 rows in a group of a workgroup's 4, or 10 in one of its 64, and then the
    # groups: below 96 (64 bits from there on); 64 u an element for xh itself
    close(dw, ref["dw"], ref["dw_tol"] * 160 / 128, "dweight")
    close(db, ref["db"], ref["db_tol"], "dbias")
    del ref, ytol
    for over in (0, 1):  # in place: the next rows' loads are in flight while a row is written
        di, xi = dy.clone(), x.clone()
        got = ops.layer_norm_bwd(di, xi, w, mean, rstd, dx=(di, xi)[over])
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)
    xi = x.clone()
    assert torch.equal(ops.layer_norm_fwd(xi, w, b, 1e-5, out=xi)[0], y)


def test_layer_norm_keeps_precision_far_from_zero(dev):
    """A row's mean 1000 times its spread: the statistics' second sum takes out what the first one's rounding left."""
    g = gen(5)
    x = torch.randn(40, 825, device=dev, generator=g) + 1000.0
    dy = torch.randn(40, 825, device=dev, generator=g)
    ref = norm_ref(x, None, None, 1e-5, dy)
    y, mean, rstd = ops.layer_norm_fwd(x)
    close(y, ref["y"], 64 * U * (ref["xh"].abs() + 1), "y")
    dx = ops.layer_norm_bwd(dy, x, None, mean, rstd)[0]
    close(dx, ref["dx"], ref["dx_tol"], "dx")


def test_layer_norm_no_rows_and_special_values(dev):
    w = torch.ones(12, device=dev)
    y, mean, rstd = ops.layer_norm_fwd(torch.empty(0, 12, device=dev), w)
    assert y.shape == (0, 12) and mean.numel() == 0
    dx, dw, db = ops.layer_norm_bwd(y, y, w, mean, rstd)
    assert dx.shape == (0, 12) and not dw.any() and not db.any()
    x = torch.randn(4, 12, device=dev)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = ops.layer_norm_fwd(x, w)[0]
    assert y[1].isnan().all() and y[2].isnan().any() and torch.isfinite(y[[0, 3]]).all()
    y, _, rstd = ops.layer_norm_fwd(torch.full((2, 12), 3.0, device=dev), w, w)  # no spread at all: the bias is left
    assert torch.equal(y, torch.ones_like(y)) and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_module(dev, dtype):
    """The nn module: leading axes, an expanded gradient, partial requires_grad; its gradients against differences."""
    g = gen(3)
    m = hnn.LayerNorm(50).to(dev)
    with torch.no_grad():
        m.weight.copy_(torch.randn(50, device=dev, generator=g))
        m.bias.copy_(torch.randn(50, device=dev, generator=g))
    x = torch.randn(3, 5, 50, device=dev, generator=g).to(dtype).requires_grad_()
    y = m(x)
    assert y.shape == x.shape and y.dtype == dtype
    y.sum().backward()  # an expanded dy of ones
    ref = norm_ref(x.detach().view(15, 50), m.weight.detach(), m.bias.detach(), m.eps, torch.ones(15, 50, device=dev))
    close(x.grad.view(15, 50), ref["dx"], ref["dx_tol"] + half(x) * (ref["dx"].abs() + ref["dx_tol"]), "dx")
    close(m.weight.grad, ref["dw"], ref["dw_tol"], "dweight")
    close(m.bias.grad, ref["db"], ref["db_tol"], "dbias")
    x2 = x.detach().transpose(0, 1)  # not contiguous, no gradient wanted for it
    m.zero_grad()
    m(x2).float().square().sum().backward()
    assert m.weight.grad is not None and x2.grad is None
    if dtype == F32:  # directional derivative by central differences, in fp32 arithmetic on both sides
        xd = x.detach().clone().requires_grad_()
        c, v = torch.randn(3, 5, 50, device=dev, generator=g), torch.randn(3, 5, 50, device=dev, generator=g)
        (m(xd) * c).sum().backward()
        h = 2.0 ** -8
        with torch.no_grad():
            num = ((m(xd + h * v).double() - m(xd - h * v).double()) * c.double()).sum() / (2 * h)
        # truncation h^2/6 f''' with |f'''| of the order of |c||v|^3, rounding 64 u |y||c| / h
        scale = float((c.double().abs() * (1 + v.double().abs()) ** 3).sum())
        assert abs(float(num) - float((xd.grad.double() * v.double()).sum())) <= scale * (8 * h * h + 64 * U / h)
    nb = hnn.LayerNorm(50, elementwise_affine=False).to(dev)
    assert torch.equal(nb(x.detach()), ops.layer_norm_fwd(x.detach())[0])


# ---------------------------------------------------------------------------------------------------------------------
# losses over sampled tokens
# ---------------------------------------------------------------------------------------------------------------------
def make_rows(M, V, dtype, seed, dev, spread=3.0):
    g = gen(seed)
    x = (torch.randn(M, V, device=dev, generator=g) * spread).to(dtype)
    t = torch.randint(0, V, (M,), device=dev, generator=g)
    best = x.float().argmax(1)
    t = torch.where(torch.rand(M, device=dev, generator=g) < 0.5, best, t)
    return x, t, g


def softmax_ref(x, t, it):
    """Log-probabilities of the targets, probabilities and the band of a log-probability: v_exp_f32's and the argument's
    roundings (2 u |log p|, at most ln V + a few on average under the softmax) and the sums' 42 u, twice over."""
    a = x.double() * it
    ls = torch.log_softmax(a, 1)
    lp = ls.gather(1, t[:, None])[:, 0]
    return lp, ls, 128 * U + 2 * U * lp.abs()


def dlogits_ref(ls, t, coef, it, band, cabs):
    """coef * it * (1[target] - p) and its band: the coefficient's (cabs times the log-probability's) and the
    probabilities' own (2 u |log p| + 64 u)."""
    p = ls.exp()
    d = -p
    d[torch.arange(len(t), device=t.device), t] += 1
    hot = torch.zeros_like(p)
    hot[torch.arange(len(t), device=t.device), t] = 1
    size = p * (64 * U + 4 * U * ls.abs().clamp(max=200)) + (p + hot) * 4 * U
    tol = it * (coef.abs()[:, None] * size + (cabs * (2 * band + 8 * U))[:, None] * (p + hot))
    return d * (coef * it)[:, None], tol + 1e-36


def check_dlogits(got, want, tol, what):
    close(got, want, tol + half(got) * (want.abs() + tol) + (2.0 ** -133 if got.dtype == BF16 else 0), what)


# sizes on both sides of every register variant: pieces of 4 (fp32) / 8 (bf16) elements, 256..1024 threads
ROW_SIZES = [(1, 1), (5, 2), (3, 7), (4, 8), (7, 9), (9, 63), (9, 71), (2, 1000), (3, 1023), (2, 1024), (2, 1025),
             (3, 2049), (2, 4097), (2, 8193), (3, 10000), (2, 16385), (2, 20001), (2, 24577), (2, 32769), (1, 40961),
             (1, 49153), (2, 50000), (1, 57345), (1, 65537), (1, 81921), (1, 98305), (1, 106497), (1, 131075)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,V", ROW_SIZES)
def test_token_logp(dev, M, V, dtype):
    x, t, g = make_rows(M, V, dtype, M * 100003 + V, dev)
    for it in (1.0, 0.7):
        logp, stats = ops.token_logp(x, t, inv_tau=it)
        it64 = float(torch.tensor(it, dtype=F32))
        lp, ls, band = softmax_ref(x, t, it64)
        close(logp, lp, band, "logp")
        coef = torch.randn(M, device=dev, generator=g)
        want, tol = dlogits_ref(ls, t, coef.double(), it64, band, torch.zeros_like(band))
        d = ops.token_logp_bwd(x, t, stats, coef, inv_tau=it)
        assert d.dtype == dtype
        check_dlogits(d, want, tol, "dlogits")
        scale = torch.tensor([0.25], device=dev)
        check_dlogits(ops.token_logp_bwd(x, t, stats, coef, inv_tau=it, scale=scale), want / 4, tol / 4, "scaled")
        dyn = torch.tensor([it], device=dev)
        assert torch.equal(ops.token_logp(x, t, dyn=dyn)[0], logp)
        xi = x.clone()
        assert torch.equal(ops.token_logp_bwd(xi, t, stats, coef, inv_tau=it, dlogits=xi), d)


def policy_ref(x, t, A, w, old, ref, lo, hi, kl, it):
    lp, ls, band = softmax_ref(x, t, it)
    A, w = A.double(), w.double()
    rho = torch.ones_like(lp) if old is None else (lp - old.double()).exp()
    cut = ((A > 0) & (rho > 1 + hi)) | ((A < 0) & (rho < 1 - lo))
    L = -torch.minimum(rho * A, rho.clamp(1 - lo, 1 + hi) * A)
    g = -torch.where(cut, 0.0, rho * A)
    cabs = torch.where(cut, 0.0, (rho * A).abs())
    if kl:
        k = ref.double() - lp
        L = L + kl * (k.exp() - k - 1)
        g = g + kl * (1 - k.exp())
        cabs = cabs + kl * (k.exp() + 1)
    live = w != 0
    z = torch.zeros_like(lp)
    out = dict(loss=torch.where(live, w * L, z).sum(), logp=torch.where(live, lp, z), band=band)
    out["loss_tol"] = float(torch.where(live, (w.abs() * ((rho * A).abs() + (kl * (k.exp() + 1) if kl else 0))
                                               * (2 * band + 8 * U)), z).sum())
    coef, cabs = torch.where(live, w * g, z), torch.where(live, w.abs() * cabs, z)
    out["d"], out["d_tol"] = dlogits_ref(ls, t, coef, it, band, cabs)
    out["d"][~live] = 0
    return out


def make_policy(M, V, dtype, seed, dev, it=1.0, dead=0.3):
    x, t, g = make_rows(M, V, dtype, seed, dev)
    lp = softmax_ref(x, t, it)[0]
    w = torch.rand(M, device=dev, generator=g) + 0.1
    if M > 1:
        w[torch.rand(M, device=dev, generator=g) < dead] = 0
        w[0] = 0.5
    d = 0.3 * torch.randn(M, device=dev, generator=g).double()
    for e in (0.8, 1.3):  # off the two borders, where the gradient jumps
        d = torch.where((d - math.log(e)).abs() < 1e-3, d + 4e-3, d)
    old = (lp - d).float()
    ref = (lp + 0.3 * torch.randn(M, device=dev, generator=g)).float()
    return x, t, torch.randn(M, device=dev, generator=g), w, old, ref


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,V", ROW_SIZES + [(40, 333), (300, 77)])
def test_policy_loss(dev, M, V, dtype):
    it = 1.25
    x, t, A, w, old, ref = make_policy(M, V, dtype, M * 31 + V, dev, it)
    for kl, o in ((0.1, old), (0.0, old), (0.1, None)):
        want = policy_ref(x, t, A, w, o, ref, 0.2, 0.3, kl, it)
        d = torch.full_like(x, float("nan"))
        loss, logp = ops.policy_loss(x, t, A, w, old_logp=o, ref_logp=ref, clip=(0.2, 0.3), kl_coef=kl, inv_tau=it,
                                     dlogits=d)
        close(logp, want["logp"], want["band"], "logp")
        assert abs(float(loss) - float(want["loss"])) <= want["loss_tol"] + 2 * U * abs(float(want["loss"])), "loss"
        check_dlogits(d, want["d"], want["d_tol"], "dlogits")
        # without the gradient, over the logits' own buffer, and through the saved statistics: the same numbers
        loss2, logp2, stats, coef = ops.policy_loss(x, t, A, w, old_logp=o, ref_logp=ref, clip=(0.2, 0.3), kl_coef=kl,
                                                    inv_tau=it, save=True)
        assert torch.equal(loss2, loss) and torch.equal(logp2, logp)
        xi = x.clone()
        ops.policy_loss(xi, t, A, w, old_logp=o, ref_logp=ref, clip=(0.2, 0.3), kl_coef=kl, inv_tau=it, dlogits=xi)
        assert torch.equal(xi, d)
        check_dlogits(ops.token_logp_bwd(x, t, stats, coef, weight=w, inv_tau=it), want["d"], want["d_tol"], "saved")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [12289, 14001, 16384])
def test_rows_of_four_pieces_a_thread(dev, V, dtype):
    """Vocabularies of 12289 to 16384 words in fp32 have a register variant of their own."""
    test_token_logp(dev, 2, V, dtype)
    test_policy_loss(dev, 3, V, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_policy_loss_is_clipped_where_the_formula_says(dev, dtype):
    """Ratios 0.5, 1, 2 with advantages of both signs and zero: which of the six are cut, and their losses."""
    V = 50
    x, t, _ = make_rows(9, V, dtype, 1, dev)
    lp = softmax_ref(x, t, 1.0)[0]
    ratio = torch.tensor([0.5, 1.0, 2.0] * 3, device=dev, dtype=torch.float64)
    A = torch.tensor([1.0] * 3 + [-1.0] * 3 + [0.0] * 3, device=dev)
    old = (lp - ratio.log()).float()
    for i in range(9):
        w = torch.zeros(9, device=dev)
        w[i] = 1
        d = torch.empty_like(x)
        loss, _ = ops.policy_loss(x, t, A, w, old_logp=old, dlogits=d)
        want = [-0.5, -1.0, -1.2, 0.8, 1.0, 2.0, 0.0, 0.0, 0.0][i]
        assert abs(float(loss) - want) <= 1e-5, i
        moves = i in (0, 1, 4, 5)  # the rest is cut, or has nothing to say
        assert bool(d[i].any()) == moves and not d[torch.arange(9, device=dev) != i].any(), i


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,extra,shift", [(333, 5, 0), (1000, 0, 1), (2050, 3, 3), (131080, 1, 1)])
def test_masked_rows_strides_and_bad_values(dev, V, extra, shift, dtype):
    """Rows of weight zero hold NaN, infinities, the type's lowest value and targets from nowhere: nothing of it shows."""
    M, inf = 8, float("inf")
    x0, t, A, w, old, ref = make_policy(M, V, dtype, V, dev)
    w[:] = torch.tensor([0.3, 0, 0.2, 0, 0, 0.1, 0, 0], device=dev)
    want = policy_ref(x0, t, A, w, old, ref, 0.2, 0.2, 0.1, 1.0)
    dead = w == 0
    bad = torch.tensor([0, float("nan"), 0, inf, -inf, 0, torch.finfo(dtype).min, inf], device=dev).to(dtype)
    x = strided(torch.where(dead[:, None], bad[:, None], x0), extra, shift)
    t2 = torch.where(dead, torch.tensor([0, -100, 0, V, 1 << 40, 0, -(1 << 60), V + 7], device=dev), t)
    nan = torch.full_like(A, float("nan"))
    A2, old2, ref2 = (torch.where(dead, nan, v) for v in (A, old, ref))
    d = strided(torch.full_like(x0, 7.0), extra, shift)
    loss, logp = ops.policy_loss(x, t2, A2, w, old_logp=old2, ref_logp=ref2, kl_coef=0.1, dlogits=d)
    close(logp, want["logp"], torch.where(dead, 0.0, want["band"]), "logp")
    assert abs(float(loss) - float(want["loss"])) <= want["loss_tol"] + 2 * U * abs(float(want["loss"])), "loss"
    check_dlogits(d, want["d"], want["d_tol"], "dlogits")
    assert not d[dead].any() and not logp[dead].any()
    flat = d.as_strided((M * (V + extra) + 8,), (1,), d.storage_offset())
    pad = torch.cat([flat[r * (V + extra) + V:(r + 1) * (V + extra)] for r in range(M)] + [flat[M * (V + extra):]])
    assert pad.isnan().all(), "written beside the rows"
    # no row left at all
    loss, logp = ops.policy_loss(x, t2, A2, torch.zeros_like(w), old_logp=old2, dlogits=d)
    assert float(loss) == 0.0 and not logp.any() and not d.any()
    # a target outside the vocabulary in a row that counts: NaN, in that row alone
    t3 = t.clone()
    t3[2] = V
    loss, logp = ops.policy_loss(x0, t3, A, w, old_logp=old, dlogits=d)
    assert loss.isnan().all() and logp[2].isnan() and d[2].isnan().all()
    assert torch.isfinite(d[[0, 1, 3, 4, 5, 6, 7]].float()).all() and torch.isfinite(logp[[0, 5]]).all()
    stats = ops.token_logp(x0, t3, w)[1]
    d = ops.token_logp_bwd(x0, t3, stats, torch.ones(M, device=dev), weight=w)
    assert d[2].isnan().all() and torch.isfinite(d[[0, 5]].float()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 20001, 140003])
@pytest.mark.parametrize("sampled_here", [True, False])
def test_policy_rows_without_a_log_probability(dev, V, sampled_here, dtype):
    """A target outside the vocabulary and a NaN logit in rows that count: NaN in the loss, in the row's log-probability and
    in every column of its gradient, on-policy (no old log-probabilities) too, fused and through autograd, on both sides
    of what a workgroup's registers hold. A token of probability zero is none of these: its ratio stays 1."""
    M = 8
    x, t, A, w, old, _ = make_policy(M, V, dtype, V, dev, dead=0.0)
    t[1], t[4] = V, -100                                       # an index behind the end, the usual ignored index
    x[6, (int(t[6]) + 1) % V] = float("nan")
    x[3, int(t[3])] = -float("inf")
    A[4] = 0.0
    bad = torch.zeros(M, dtype=torch.bool, device=dev)
    bad[[1, 4, 6]] = True
    kw = dict(old_logp=None if sampled_here else old)
    for only in (None, 1, 4, 6):                               # all rows, and each of the bad ones alone
        wi = w if only is None else torch.where(torch.arange(M, device=dev) == only, w, 0.0)
        hit = bad & (wi != 0)
        d = torch.empty_like(x)
        loss, logp = ops.policy_loss(x, t, A, wi, dlogits=d, **kw)
        xr = x.clone().requires_grad_()
        loss2, logp2 = hnn.policy_loss(xr, t, A, wi, **kw)
        loss2.backward()
        assert loss.isnan().all() and loss2.isnan(), only
        for lp, grad in ((logp, d), (logp2, xr.grad)):
            assert torch.equal(lp.isnan(), hit), only
            assert grad[hit].isnan().all() and torch.isfinite(grad[~hit].float()).all(), only
    wi = torch.where(bad, 0.0, w)                              # without them
    loss, logp = ops.policy_loss(x, t, A, wi, **kw)
    assert torch.isfinite(loss).all() and float(logp[3]) == -float("inf")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [40, 3000, 140000])
def test_banned_tokens(dev, V, dtype):
    """-inf and the type's lowest value in rows that count: those tokens have probability and gradient zero."""
    x, t, A, w, old, ref = make_policy(6, V, dtype, V, dev, dead=0.0)
    keep = torch.zeros(6, V, dtype=torch.bool, device=dev)
    keep[torch.arange(6, device=dev), t] = True
    ban = (torch.rand(6, V, device=dev, generator=gen(9)) < 0.5) & ~keep
    ban[5] = ~keep[5]  # everything but the target
    x[ban] = -float("inf")
    x[:3][ban[:3]] = torch.finfo(dtype).min
    want = policy_ref(x, t, A, w, None, ref, 0.2, 0.2, 0.0, 1.0)
    d = torch.empty_like(x)
    loss, logp = ops.policy_loss(x, t, A, w, dlogits=d)
    close(logp, want["logp"], want["band"], "logp")
    assert float(logp[5]) == 0.0 and not d[5].any()
    assert not d[ban].any() and torch.isfinite(d.float()).all()
    want["d"][ban], want["d_tol"][ban] = 0, 0
    check_dlogits(d, want["d"], want["d_tol"], "dlogits")
    y = x.clone()
    y[2, int(t[2]) - 1] = float("inf")  # an infinite logit: NaN, in its row alone
    _, logp = ops.policy_loss(y, t, A, w, dlogits=d)
    assert logp[2].isnan() and d[2].isnan().all() and torch.isfinite(logp[[0, 1, 3, 4, 5]]).all()
    x[1] = -float("inf")  # no token is possible: as log_softmax says, NaN
    _, logp = ops.policy_loss(x, t, A, w, dlogits=d)
    assert logp[1].isnan() and d[1].isnan().all() and torch.isfinite(logp[[0, 2, 3, 4, 5]]).all()
    _, logp = ops.policy_loss(x, t, A, w)
    assert logp[1].isnan()


def test_kl_of_a_banned_target_is_infinite(dev):
    """e^k - k - 1 grows without bound as the token's probability goes to zero: infinity, and no NaN from inf - inf."""
    x, t, A, w, old, ref = make_policy(6, 300, F32, 11, dev, dead=0.0)
    x[2, t[2]] = -float("inf")
    for weight in (w, w * (torch.arange(6, device=dev) != 2)):
        loss, logp = ops.policy_loss(x, t, A, weight, ref_logp=ref, kl_coef=0.1)
        assert torch.isfinite(loss) if float(weight[2]) == 0 else float(loss) == float("inf")
    loss, logp = ops.policy_loss(x, t, A, w, ref_logp=ref, kl_coef=0.0)  # -lp A alone is no part of the loss: rho = 1
    assert torch.isfinite(loss) and float(logp[2]) == -float("inf")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [37, 5001, 140003])
@pytest.mark.parametrize("base", [-3.0e38, -1.0e30, -2.0e6, 1.0e5, 2.0e6, 1.0e30, 3.0e38])
def test_rows_far_from_zero(dev, V, base, dtype):
    """Rows all of whose logits are at one far value (a mask's lowest value among them), and rows spread around it: the
    log-probabilities are those of the differences, which are exact here."""
    x = torch.full((3, V), base, device=dev).to(dtype)
    step = float(torch.nextafter(x[0, 0], torch.zeros((), device=dev, dtype=dtype))) - float(x[0, 0])
    g = gen(V)
    n = torch.randint(0, 3, (V,), device=dev, generator=g)
    x[1] = (x[1].double() + step * n.double()).to(dtype)  # one, two or three neighbouring values
    x[2, : V // 2] = torch.finfo(dtype).min
    t = torch.tensor([0, int(n.argmax()), V - 1], device=dev)
    lp, ls, band = softmax_ref(x, t, 1.0)
    # a row's differences are exact, so only the exponentials' own roundings are left: |difference| * 2 u each
    band = 128 * U + 4 * U * lp.abs()
    logp, stats = ops.token_logp(x, t)
    close(logp, lp, band + torch.where(lp.abs() > 80, 2 * U * lp.abs(), 0.0), "logp")
    coef = torch.ones(3, device=dev)
    want, tol = dlogits_ref(ls, t, coef.double(), 1.0, band, torch.zeros_like(band))
    tol = tol + 128 * U * ls.exp()
    check_dlogits(ops.token_logp_bwd(x, t, stats, coef), want, tol, "dlogits")
    d = torch.empty_like(x)
    ops.policy_loss(x, t, -coef, dlogits=d)
    check_dlogits(d, want, tol, "dlogits of the fused pass")


def pair_ref(x, t, w, ref, beta, smooth, it):
    P = w.shape[0] // 2
    lp, ls, band = softmax_ref(x, t, it)
    w64 = w.double()
    live = w64 != 0
    z = torch.zeros_like(w64)
    S = torch.where(live, w64 * lp.view_as(w64), z).sum(1)
    dS = torch.where(live, w64.abs() * band.view_as(w64), z).sum(1)
    gain = S - ref.double()
    m = beta * (gain[:P] - gain[P:])
    dm = beta * (dS[:P] + dS[P:])
    loss = -((1 - smooth) * torch.nn.functional.logsigmoid(m) + smooth * torch.nn.functional.logsigmoid(-m))
    up = -(beta / P) * ((1 - smooth) * torch.sigmoid(-m) - smooth * torch.sigmoid(m))
    dup = beta / P * (dm / 4 + 4 * U * up.abs())
    coef = (torch.cat((up, -up))[:, None] * w64).view(-1)
    cerr = (torch.cat((dup, dup))[:, None] * w64.abs()).view(-1)
    d, tol = dlogits_ref(ls, t, coef, it, torch.zeros_like(band), coef.abs() + 1)
    hot = torch.zeros_like(d)
    hot[torch.arange(len(t), device=t.device), t] = 1
    tol = tol + it * (cerr + 4 * U * coef.abs())[:, None] * (ls.exp() + hot)
    d[~live.view(-1)] = 0
    return dict(S=S, dS=dS + U * S.abs(), m=m, dm=dm + U * m.abs(), loss=loss.mean(), dl=float(dm.mean()), d=d, tol=tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,T,V", [(1, 1, 5), (1, 3, 1000), (3, 1, 33), (2, 65, 77), (5, 21, 300), (2, 7, 20001),
                                   (1, 2, 131075), (70, 3, 40), (70, 65, 9), (9, 2, 300), (600, 1, 12), (2100, 1, 5)])
def test_preference_loss(dev, P, T, V, dtype):
    x, t, g = make_rows(2 * P * T, V, dtype, P * 1009 + T * 101 + V, dev)
    n = torch.randint(0, T + 1, (2 * P, 1), device=dev, generator=g)
    n[0] = T
    w = (torch.arange(T, device=dev)[None] < n).float() * (1 + torch.rand(2 * P, T, device=dev, generator=g))
    if P > 1:
        w[1] = 0  # an empty sentence
    S = (softmax_ref(x, t, 1.0)[0].view(2 * P, T) * w).sum(1)
    ref = (S + 5 * torch.randn(2 * P, device=dev, generator=g)).float()
    x = torch.where((w.view(-1) == 0)[:, None], torch.full_like(x, float("nan")), x)
    xr = torch.nan_to_num(x)
    for smooth, it in ((0.0, 1.0), (0.2, 0.5)):
        want = pair_ref(xr, t, w, ref, 0.3, smooth, it)
        d = torch.full_like(x, float("nan"))
        loss, margin, seq = ops.preference_loss(x, t, w, ref, beta=0.3, label_smoothing=smooth, inv_tau=it, dlogits=d)
        close(seq, want["S"], want["dS"], "seq_logp")
        close(margin, want["m"], want["dm"], "margin")
        assert abs(float(loss) - float(want["loss"])) <= want["dl"] + 2 * U * abs(float(want["loss"])), "loss"
        check_dlogits(d, want["d"], want["tol"], "dlogits")
        l2, m2, s2 = ops.preference_loss(x, t, w, ref, beta=0.3, label_smoothing=smooth, inv_tau=it)
        assert torch.equal(l2, loss) and torch.equal(m2, margin) and torch.equal(s2, seq)
        xi = x.clone()
        ops.preference_loss(xi, t, w, ref, beta=0.3, label_smoothing=smooth, inv_tau=it, dlogits=xi)
        assert torch.equal(xi, d)


def test_preference_loss_far_margins(dev):
    """Margins of +-1000: the loss is the margin or zero, nothing overflows."""
    x, t, _ = make_rows(4, 20, F32, 3, dev)
    w = torch.ones(4, 1, device=dev)
    ref = torch.tensor([-1000.0, 1000.0, 1000.0, -1000.0], device=dev)
    d = torch.empty_like(x)
    loss, margin, _ = ops.preference_loss(x, t, w, ref, beta=1.0, dlogits=d)
    assert 1900 < float(margin[0]) < 2100 and -2100 < float(margin[1]) < -1900
    assert abs(float(loss) + float(margin[1]) / 2) <= 1e-3
    assert not d[0].any() and not d[2].any() and torch.isfinite(d).all() and d[1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,T,V", [(1, 1, 40), (3, 4, 3000), (12, 2, 300), (3, 1, 140003)])
def test_preference_loss_of_impossible_sentences(dev, P, T, V, dtype):
    """A sentence with a banned word (logit -inf) has log-probability -inf. Rejected, its pair is decided: margin +inf, loss
    -log sigmoid(inf) = 0 and no gradient without smoothing, +inf with it. Chosen: margin -inf, loss +inf. The gradients
    are finite: sigmoid(+-inf) is 0 or 1. The other pairs' numbers are as without it."""
    x, t, g = make_rows(2 * P * T, V, dtype, 17 * P + V, dev)
    w = 1 + torch.rand(2 * P, T, device=dev, generator=g)
    S = (softmax_ref(x, t, 1.0)[0].view(2 * P, T) * w).sum(1)
    ref = (S + 3 * torch.randn(2 * P, device=dev, generator=g)).float()
    odd, beta, inf = P - 1, 0.3, float("inf")
    rest = [p for p in range(P) if p != odd]
    sents = rest + [P + p for p in rest]
    for side, smooth in ((1, 0.0), (1, 0.1), (0, 0.0), (0, 0.1)):
        xb = x.clone()
        row = (side * P + odd) * T + T // 2
        xb[row, int(t[row])] = -inf
        d = torch.full_like(x, float("nan"))
        loss, margin, seq = ops.preference_loss(xb, t, w, ref, beta=beta, label_smoothing=smooth, dlogits=d)
        alone = ops.preference_loss(xb, t, w, ref, beta=beta, label_smoothing=smooth)
        assert all(torch.equal(a, b) for a, b in zip(alone, (loss, margin, seq)))
        assert float(margin[odd]) == (inf if side else -inf) and float(seq[side * P + odd]) == -inf
        total, band = 0.0, 0.0
        if rest:
            pick = torch.tensor([s * T + i for s in sents for i in range(T)], device=dev)
            want = pair_ref(x[pick], t[pick], w[sents], ref[sents], beta, smooth, 1.0)
            f = len(rest) / P
            total, band = float(want["loss"]) * f, want["dl"] * f
            check_dlogits(d[pick], want["d"] * f, want["tol"] * f, "the other pairs' dlogits")
        if side and not smooth:
            assert abs(float(loss) - total) <= band + 2 * U * abs(total), (side, smooth)
        else:
            assert float(loss) == inf, (side, smooth)
        # d loss / dS of the chosen sentence, minus that of the rejected one
        up = beta / P * smooth if side else -beta / P * (1 - smooth)
        own = torch.tensor([s * T + i for s in (odd, P + odd) for i in range(T)], device=dev)
        _, ls, _ = softmax_ref(xb[own], t[own], 1.0)
        coef = (w[[odd, P + odd]].double() * torch.tensor([[up], [-up]], device=dev)).view(-1)
        want, tol = dlogits_ref(ls, t[own], coef, 1.0, torch.zeros_like(coef), coef.abs())
        check_dlogits(d[own], want, tol, "dlogits of the pair")
        if up == 0:
            assert not d[own].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_loss_modules(dev, dtype):
    """The differentiable forms: the gradient times the upstream one, and (fp32) against differences."""
    M, V = 12, 301
    x, t, A, w, old, ref = make_policy(M, V, dtype, 8, dev)
    kw = dict(old_logp=old, ref_logp=ref, kl_coef=0.1)
    d = torch.empty_like(x)
    loss0, logp0 = ops.policy_loss(x, t, A, w, dlogits=d, **kw)
    xr = x.clone().requires_grad_()
    loss, logp = hnn.policy_loss(xr, t, A, w, **kw)
    assert loss.dim() == 0 and torch.equal(loss.detach(), loss0[0]) and torch.equal(logp, logp0) and not logp.requires_grad
    (2.0 * loss).backward()
    want = policy_ref(x, t, A, w, old, ref, 0.2, 0.2, 0.1, 1.0)
    check_dlogits(xr.grad, 2 * want["d"], 2 * want["d_tol"], "policy dlogits")
    pw = w.view(4, 3)
    sref = torch.randn(4, device=dev, generator=gen(1)) * 3 - 20
    ploss, margin, seq = hnn.preference_loss(xr, t, pw, sref, beta=0.2)
    xr.grad = None
    ploss.backward()
    pwant = pair_ref(x, t, pw, sref, 0.2, 0.0, 1.0)
    check_dlogits(xr.grad, pwant["d"], pwant["tol"], "preference dlogits")
    if dtype != F32:
        return
    h = 2.0 ** -7
    v = torch.randn(M, V, device=dev, generator=gen(2))
    v = v / v.norm()
    slope = lambda f: float(f(x + h * v).double() - f(x - h * v).double()) / (2 * h)  # noqa: E731
    for f, grad in ((lambda z: ops.preference_loss(z, t, pw, sref, beta=0.2)[0], xr.grad),
                    (lambda z: ops.policy_loss(z, t, A, w, clip=(0.9, 9.0), **kw)[0], None)):
        if grad is None:  # (bounds that no ratio reaches: smooth)
            grad = torch.empty_like(x)
            ops.policy_loss(x, t, A, w, clip=(0.9, 9.0), dlogits=grad, **kw)
        # |v| = 1: third derivatives are of the order of the weights' sum; rounding 256 u sum(w |lp|) / h
        assert abs(slope(f) - float((grad.double() * v.double()).sum())) <= 30 * float(w.sum()) * (h * h + 64 * U / h)


@pytest.mark.parametrize("form", ["policy", "preference"])
def test_losses_take_in_place_arithmetic(dev, form):
    """What a training loop does with a loss, loss /= steps and loss += another one, and with the numbers beside it: they
    are tensors of their own, from the differentiable forms and from the explicit ones."""
    M, V = 12, 40
    x, t, A, w, old, _ = make_policy(M, V, F32, 5, dev, dead=0.0)
    sref = torch.zeros(4, device=dev)

    def call(m, v):
        return m.policy_loss(v, t, A, w, old_logp=old) if form == "policy" else m.preference_loss(v, t, w.view(4, 3), sref,
                                                                                                   beta=0.2)

    plain = x.clone().requires_grad_()
    loss = call(hnn, plain)[0] / 4
    (loss + plain.square().mean()).backward()
    xr = x.clone().requires_grad_()
    got = call(hnn, xr)
    beside = [b.clone() for b in got[1:]]
    total = got[0]
    total /= 4
    total += xr.square().mean()
    for b in got[1:]:
        b.mul_(2.0)
    total.backward()
    assert torch.equal(total.detach(), (loss + plain.square().mean()).detach())
    close(xr.grad, plain.grad, 2 * U * plain.grad.double().abs(), "gradient")  # (the two parts may be added in either order)
    assert all(torch.equal(b, 2 * k) for b, k in zip(got[1:], beside))
    explicit = call(ops, x)
    aux = torch.ones((), device=dev, requires_grad=True)
    total = explicit[0]
    total += aux
    total.sum().backward()
    assert float(aux.grad) == 1.0 and not any(b.requires_grad for b in explicit[1:])


def test_long_offsets(dev):
    """More than 2^31 elements of logits: the last rows are read and written where they are."""
    V, M = 50000, 43100
    x = torch.zeros(M, V, device=dev, dtype=BF16)
    tail, t, A, _, old, ref = make_policy(3, V, BF16, 4, dev)
    x[-3:] = tail
    target = torch.zeros(M, dtype=torch.int64, device=dev)
    target[-3:] = t
    w, adv = torch.zeros(M, device=dev), torch.zeros(M, device=dev)
    w[-3:], adv[-3:] = 1.0, A
    want = policy_ref(tail, t, A, torch.ones(3, device=dev), None, None, 0.2, 0.2, 0.0, 1.0)
    d = torch.full_like(x, 5.0)
    loss, logp = ops.policy_loss(x, target, adv, w, dlogits=d)
    close(logp[-3:], want["logp"], want["band"], "logp")
    check_dlogits(d[-3:], want["d"], want["d_tol"], "dlogits")
    assert not d[:-3].any()
    _, stats = ops.token_logp(x, target, w)
    coef = torch.zeros(M, device=dev)
    coef[-3:] = -A
    d.fill_(5.0)
    ops.token_logp_bwd(x, target, stats, coef, weight=w, dlogits=d)
    check_dlogits(d[-3:], want["d"], want["d_tol"], "dlogits, second pass")
    assert not d[:-3].any()


def test_more_rows_than_a_grid_holds(dev):
    """2^31 threads are the most of one launch: the rows behind that take another one."""
    M, V = (1 << 23) + 5, 3
    x = torch.randn(M, V, device=dev, generator=gen(6))
    t = torch.randint(0, V, (M,), device=dev, generator=gen(7))
    A = torch.randn(M, device=dev, generator=gen(8))
    w = (torch.rand(M, device=dev, generator=gen(9)) < 0.9).float() / M
    d = torch.empty_like(x)
    loss, logp = ops.policy_loss(x, t, A, w, dlogits=d)
    want = policy_ref(x, t, A, w, None, None, 0.2, 0.2, 0.0, 1.0)
    close(logp, want["logp"], want["band"], "logp")
    assert abs(float(loss) - float(want["loss"])) <= want["loss_tol"] + 2 * U * abs(float(want["loss"]))
    check_dlogits(d, want["d"], want["d_tol"], "dlogits")


def test_more_pairs_than_a_grid_holds(dev):
    """2^25 pairs and some of one token each, at 128 threads a pair: more than one launch of the pair kernel."""
    P, V, beta = (1 << 25) + 3, 2, 0.5
    x = torch.randn(2 * P, V, device=dev, generator=gen(1))
    t = torch.randint(0, V, (2 * P,), device=dev, generator=gen(2))
    w = torch.rand(2 * P, 1, device=dev, generator=gen(3)) + 0.5
    ref = torch.randn(2 * P, device=dev, generator=gen(4))
    d = torch.full_like(x, float("nan"))
    loss, margin, seq = ops.preference_loss(x, t, w, ref, beta=beta, dlogits=d)
    lp, ls, band = softmax_ref(x, t, 1.0)
    S, dS = lp * w[:, 0].double(), band * w[:, 0].double()
    close(seq, S, dS + U * S.abs(), "seq_logp")
    gain = S - ref.double()
    m, dm = beta * (gain[:P] - gain[P:]), beta * (dS[:P] + dS[P:])
    close(margin, m, dm + U * m.abs(), "margin")
    want = float(-torch.nn.functional.logsigmoid(m).mean())
    assert abs(float(loss) - want) <= float(dm.mean()) + 2 * U * want
    up, dup = -(beta / P) * torch.sigmoid(-m), beta / P * dm / 4
    coef, cerr = torch.cat((up, -up)) * w[:, 0].double(), torch.cat((dup, dup)) * w[:, 0].double()
    wd, tol = dlogits_ref(ls, t, coef, 1.0, torch.zeros_like(band), coef.abs())
    check_dlogits(d, wd, tol + 2 * cerr[:, None], "dlogits")  # (p + 1 at the target is at most 2)


# ---------------------------------------------------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------------------------------------------------
def grads_of(sizes, dev, seed=0, mixed=True):
    g = gen(seed)
    return [torch.randn(*s, device=dev, generator=g).to(BF16 if mixed and i % 3 == 1 else F32)
            for i, s in enumerate(sizes)]


def norm64(grads, kind=2.0):
    v = torch.cat([t.reshape(-1).double() for t in grads])
    return float(v.norm()) if kind == 2.0 else float(v.abs().max())


SHAPES = [(7,), (300, 12), (1,), (825, 33), (4096,), (4097,), (0,), (3, 5, 7), (100000,), (64, 64), (513, 257)]


def check_clipped(got, grads, norm, want_norm, max_norm, scale=1.0):
    assert abs(float(norm) - want_norm) <= 2 * U * want_norm
    f = scale * min(1.0, max_norm / (want_norm + 1e-6))
    for o, g in zip(got, grads):
        w = g.double() * f
        close(o, w, w.abs() * (half(g) + 4 * U) + (2.0 ** -133 if g.dtype == BF16 else 2.0 ** -149), "clipped")


@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6, float("inf")])
def test_clip(dev, kind, max_norm):
    grads = grads_of(SHAPES, dev)
    keep = [g.clone() for g in grads]
    want = norm64(grads, kind)
    assert abs(float(ops.grad_norm(grads, kind)) - want) <= 2 * U * want
    out = [torch.full_like(g, 9.0) for g in grads]
    check_clipped(out, keep, ops.clip_grad_norm(grads, max_norm, kind, out=out), want, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    norm = ops.clip_grad_norm(grads, max_norm, kind)
    check_clipped(grads, keep, norm, want, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))
    assert max_norm < 1 or all(torch.equal(a, b) for a, b in zip(grads, keep))


@pytest.mark.parametrize("count", [1, 71, 72, 73, 150, 300])
def test_clip_many_tensors(dev, count):
    grads = grads_of([((i * 37) % 900 + 1,) if i % 2 else (i % 7 + 1, (i * 13) % 300 + 1) for i in range(count)], dev, count)
    keep = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, 1.5, grad_scale=0.25)
    want = 0.25 * norm64(keep)
    check_clipped(grads, keep, norm, want, 1.5, 0.25)
    assert torch.equal(ops.grad_norm(keep, grad_scale=-0.25), norm)


@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("sizes", [[(5000001,), (1234567,), (3,), (1999, 1501), (0,), (70001,)],
                                   [(17000003,), (8193,), (16900001,), (4000, 1023), (2,), (300, 12)]])
def test_clip_large_lists(dev, sizes, kind):
    """More elements than the smallest share of a workgroup leaves to 1024 of them (every thread makes several trips), and
    more than 32 M (written past the caches); sizes off the shares, mixed types, one matrix with a row stride."""
    grads = grads_of(sizes, dev, len(sizes))
    wide = torch.randn(sizes[3][0], sizes[3][1] + 5, device=dev, generator=gen(3))
    grads[3] = wide[:, :sizes[3][1]]
    keep, gap = [t.clone() for t in grads], wide[:, sizes[3][1]:].clone()
    want = norm64(grads, kind)
    out = [torch.full_like(t, 9.0) for t in keep]
    out[3] = torch.full_like(wide, 9.0)[:, :sizes[3][1]]
    norm = ops.clip_grad_norm(grads, want / 8, kind, out=out)
    check_clipped(out, keep, norm, want, want / 8)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    assert torch.equal(ops.clip_grad_norm(grads, want / 8, kind), norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out)) and torch.equal(wide[:, sizes[3][1]:], gap)


def test_clip_layouts(dev):
    """Padded matrix views, permuted pieces, odd starts; what lies between the rows stays as it is."""
    g = gen(2)
    buf = torch.randn(40000, device=dev, generator=g)
    b16 = torch.randn(40000, device=dev, generator=g).to(BF16)
    views = [buf[1:1 + 20 * 828].view(20, 828)[:, :825], buf[17000:17000 + 12].view(3, 4).t(),
             buf[18001:18001 + 30 * 31].view(30, 31)[:, 1:30], buf[20001:20008],
             buf[21000:21000 + 9000 * 2].view(9000, 2)[:, :1], buf[39100:39100 + 100 * 9].view(100, 9)[:, 2:5],
             b16[3:3 + 50 * 130].view(50, 130)[:, :129], b16[7001:7001 + 60].view(5, 4, 3).permute(2, 0, 1)]
    keep, bkeep, gk = buf.clone(), b16.clone(), [v.clone() for v in views]
    want = norm64(views)
    norm = ops.clip_grad_norm(views, 3.0)
    check_clipped(views, gk, norm, want, 3.0)
    for v, k in ((buf, keep), (b16, bkeep)):
        for a in [q for q in views if q.dtype == v.dtype]:
            off = (a.data_ptr() - v.data_ptr()) // v.element_size()
            a.copy_(k.as_strided(a.shape, a.stride(), off))
        assert torch.equal(v, k), "written outside the views"
    out = [torch.empty(20, 900, device=dev)[:, :825], torch.empty(4, 3, device=dev).t().contiguous().t()]
    got = ops.clip_grad_norm([views[0], torch.randn(4, 3, device=dev).t().contiguous().t()], 1.0, out=out)
    assert torch.isfinite(got).all()


def test_norm_of_extreme_values(dev):
    """Squares that fp32 cannot hold, and squares that vanish in it: the sum is formed in 64 bits."""
    big, small = torch.full((1000,), 1e30, device=dev), torch.full((1000,), 1e-30, device=dev)
    for t, v in ((big, 1e30), (small, 1e-30)):
        want = math.sqrt(1000) * float(torch.tensor(v, dtype=F32))
        assert abs(float(ops.grad_norm([t])) - want) <= 2 * U * want
    ops.clip_grad_norm([big], 1.0)
    assert abs(float(big.double().norm()) - 1.0) <= 1e-6
    for bad in (float("nan"), float("inf")):
        t = torch.ones(5000, device=dev)
        t[4321] = bad
        n, m = ops.grad_norm([t]), ops.grad_norm([t], float("inf"))
        assert (n.isnan() and m.isnan()) if bad != bad else (n.isinf() and m.isinf())
        u = torch.ones(3, device=dev)
        ops.clip_grad_norm([t, u], 1.0)
        ref = torch.ones(3) * torch.clamp(torch.tensor(1.0) / (torch.tensor(bad) + 1e-6), max=1.0)
        assert torch.equal(u.cpu().nan_to_num(7.0), ref.nan_to_num(7.0))
        assert t[4321].isnan()
    assert float(ops.grad_norm([torch.zeros(10, device=dev)])) == 0.0
    assert float(ops.grad_norm([torch.zeros(0, device=dev)])) == 0.0
    assert float(ops.clip_grad_norm([torch.zeros(0, device=dev)], 1.0)) == 0.0


def test_clip_parameters(dev):
    """nn.clip_grad_norm_ on modules, beside torch's own on copies of the same gradients."""
    lin = hnn.Linear(33, 20).to(dev)
    ln = hnn.LayerNorm(33).to(dev)
    unused = torch.nn.Parameter(torch.zeros(3, device=dev))
    y = lin(ln(torch.randn(9, 33, device=dev, generator=gen(1))))
    (y * y).sum().backward()
    params = list(lin.parameters()) + [unused] + list(ln.parameters())
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, twin):
        q.grad = None if p.grad is None else p.grad.clone()
    n0 = torch.nn.utils.clip_grad_norm_(twin, 0.7)
    n1 = hnn.clip_grad_norm_(params, 0.7)
    assert abs(float(n0) - float(n1)) <= 64 * U * float(n0)
    for p, q in zip(params, twin):
        assert (p.grad is None) == (q.grad is None)
        if p.grad is not None:
            close(p.grad, q.grad, 64 * U * q.grad.double().abs(), "clipped")
    assert float(hnn.clip_grad_norm_([unused], 1.0)) == 0.0


@pytest.mark.parametrize("n", [1, 5, 4099, 300001, 1 << 20, (1 << 20) + 1, 33554433])
def test_adam_clipped(dev, n):
    g = gen(n)
    mk = lambda s=1.0: s * torch.randn(n, device=dev, generator=g)  # noqa: E731
    p, grad, m, v = mk(), mk(), mk(0.1), mk().square()
    want = norm64([grad]) * 0.5
    for max_norm in (0.3, 1e9):
        a, b = [[t.clone() for t in (p, m, v)] for _ in range(2)]
        norm = ops.adam(a[0], grad, a[1], a[2], 1e-2, 7, grad_scale=0.5, max_norm=max_norm)
        assert abs(float(norm) - want) <= 2 * U * want
        c = min(1.0, max_norm / (want + 1e-6))
        ops.adam(b[0], grad, b[1], b[2], 1e-2, 7, grad_scale=0.5 * c)
        for x, y, s in zip(a, b, (p, m, v)):  # (the two scales differ by a rounding; the update is at most a few lr)
            close(x, y, 16 * U * (y.double().abs() + s.double().abs() + 1e-2), "adam")
        if c == 1.0:
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert ops.adam(p, grad, m, v, 1e-2, 7) is None


def test_adam_of_streamed_arenas(dev):
    """Arenas of 32 M elements and more pass the caches by: the update against its formula in 64 bits, and bit for bit
    against the same arena updated in slices below that size."""
    n, step, gs = (32 << 20) + 4103, 7, 0.5
    g = gen(1)
    p, grad, m, v = [torch.randn(n, device=dev, generator=g) for _ in range(4)]
    m, v = m * 0.1, v.square()
    f = lambda x: float(torch.tensor(x, dtype=F32))  # noqa: E731
    lr, b1, b2, eps = f(1e-2), f(0.9), f(0.999), f(1e-8)
    a, b = [[t.clone() for t in (p, m, v)] for _ in range(2)]
    assert ops.adam(a[0], grad, a[1], a[2], 1e-2, step, grad_scale=gs) is None
    for lo, hi in ((0, 12 << 20), (12 << 20, (25 << 20) + 4), ((25 << 20) + 4, n)):  # (16-byte aligned, odd end)
        ops.adam(b[0][lo:hi], grad[lo:hi], b[1][lo:hi], b[2][lo:hi], 1e-2, step, grad_scale=gs)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    p64, g64, m64, v64 = p.double(), grad.double() * gs, m.double(), v.double()
    mw = m64 + (g64 - m64) * (1 - b1)
    # three roundings of the difference's term, one of the sum
    mtol = U * (4 * (g64 - m64).abs() * (1 - b1) + mw.abs())
    close(a[1], mw, mtol, "m")
    vw = b2 * v64 + (1 - b2) * g64 * g64
    close(a[2], vw, 5 * U * vw, "v")
    den = vw.sqrt() / (1 - b2 ** step) ** 0.5 + eps
    upd = lr / (1 - b1 ** step) * mw / den
    # the root of 5 u, its own, the corrections' (1 each), two divisions, a sum, two products: below 12 u
    close(a[0], p64 - upd, 12 * U * upd.abs() + lr / (1 - b1 ** step) * mtol / den + U * (p64 - upd).abs() + 2 * U * upd.abs(),
          "p")
    clipped = [t.clone() for t in (p, m, v)]
    norm = ops.adam(clipped[0], grad, clipped[1], clipped[2], 1e-2, step, grad_scale=gs, max_norm=float("inf"))
    assert all(torch.equal(x, y) for x, y in zip(a, clipped))
    want = norm64([grad]) * gs
    assert abs(float(norm) - want) <= 2 * U * want


def test_arena_step_is_clipped(dev):
    """AdamState.apply(max_norm=...): padded views and fused groups; the padding adds nothing to the norm."""
    torch.manual_seed(0)
    named = [("a", torch.nn.Parameter(torch.randn(70, 825))), ("b", torch.nn.Parameter(torch.randn(11))),
             ("c", torch.nn.Parameter(torch.randn(66, 70)))]
    arenas = [ParamArena([(n, torch.nn.Parameter(p.detach().clone().to(dev))) for n, p in named], dev) for _ in range(2)]
    g = [torch.randn(p.shape, device=dev, generator=gen(4)) for _, p in named]
    for a in arenas:
        for (n, _), t in zip(named, g):
            a.grads[n].copy_(t)
    want = norm64(g)
    norm = arenas[0].new_adam().apply(1e-3, max_norm=want / 8)
    assert abs(float(norm) - want) <= 2 * U * want
    ops.clip_grad_norm(list(arenas[1].grads.values()), want / 8)
    arenas[1].new_adam().apply(1e-3)
    close(arenas[0].p, arenas[1].p, 1e-3 * 64 * U + 4 * U * arenas[1].p.double().abs(), "p")
    st = arenas[0].new_adam()
    st.sync_device_step()
    assert abs(float(st.apply(1e-3, dynamic=True, max_norm=1.0)) - want) <= 2 * U * want


# ---------------------------------------------------------------------------------------------------------------------
# together, on streams, in graphs
# ---------------------------------------------------------------------------------------------------------------------
def tune_step(ln, fc, h, t, A, w, old):
    """Hidden states -> layer norm -> vocabulary projection -> policy loss -> gradients -> clipping."""
    params = list(ln.parameters()) + list(fc.parameters())
    for p in params:
        p.grad = None
    logits = fc(ln(h))
    loss, _ = hnn.policy_loss(logits, t, A, w, old_logp=old)
    loss.backward()
    norm = hnn.clip_grad_norm_(params, 0.05)
    return loss.detach(), norm, [p.grad for p in params]


def test_chain(dev):
    """The operators as a tuning step uses them, against the same chain in 64-bit torch on the CPU."""
    torch.manual_seed(1)
    M, H, V = 42, 60, 500
    ln, fc = hnn.LayerNorm(H).to(dev), hnn.Linear(H, V).to(dev)
    h = torch.randn(M, H, device=dev, generator=gen(1)).requires_grad_()
    t = torch.randint(0, V, (M,), device=dev, generator=gen(2))
    A = torch.randn(M, device=dev, generator=gen(3))
    w = (torch.rand(M, device=dev, generator=gen(4)) < 0.7).float() / M
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in (ln.weight, ln.bias, fc.weight, fc.bias)]
    hr = h.detach().double().cpu().requires_grad_()
    z = torch.nn.functional.layer_norm(hr, (H,), ref[0], ref[1]) @ ref[2].t() + ref[3]
    lp = torch.log_softmax(z, 1).gather(1, t.cpu()[:, None])[:, 0]
    old = (lp.detach() - 0.02 * torch.randn(M, generator=torch.Generator().manual_seed(5))).float()
    rho = (lp - old.double()).exp()
    Ad, wd = A.double().cpu(), w.double().cpu()
    loss = -(wd * torch.minimum(rho * Ad, rho.clamp(0.8, 1.2) * Ad)).sum()
    loss.backward()
    norm = torch.nn.utils.clip_grad_norm_(ref, 0.05)
    got_loss, got_norm, grads = tune_step(ln, fc, h, t, A, w, old.to(dev))
    # fp32 products of H = 60 and M = 42 terms behind the operators' own roundings
    assert abs(float(got_loss) - float(loss)) <= 1e-6 and abs(float(got_norm) - float(norm)) <= 1e-5 * float(norm)
    for g, r in zip(grads + [h.grad], [p.grad for p in ref] + [hr.grad]):
        assert (g.double().cpu() - r).norm() <= 1e-5 * r.norm()


@pytest.mark.parametrize("form", ["policy", "preference"])
def test_gradients_into_the_generator(dev, form):
    """The losses behind the framework's own generator: gradients of its LSTM and projection, of the words and of the code
    against the same model in 64-bit torch on the CPU."""
    from ldrs_amd.model.generator import Generator
    from ldrs_amd.utils.config import Config
    torch.manual_seed(3)
    cfg = Config(7, 5, 50, 20, 1e-3, 7.9, 0.1, 0.1, 1.0, word_embed_size=12, latent_variable_size=6, decoder_rnn_size=20)
    B, T, V, E, Z = 6, 7, 50, 12, 7
    net = Generator(cfg).to(dev)
    words = torch.randn(B, T, E, device=dev, generator=gen(1)).requires_grad_()
    code = torch.randn(B, Z, device=dev, generator=gen(2)).requires_grad_()
    t = torch.randint(0, V, (B * T,), device=dev, generator=gen(3))
    A = torch.randn(B * T, device=dev, generator=gen(4))
    w = (torch.arange(T, device=dev)[None] < torch.tensor([[7], [5], [7], [1], [6], [3]], device=dev)).float()
    shift = 0.05 * torch.randn(B * T, device=dev, generator=gen(5))
    sref = -20 + torch.randn(B, device=dev, generator=gen(6))

    rnn = torch.nn.LSTM(E + Z, 20, num_layers=2, batch_first=True).double()
    rnn.load_state_dict({k: v.double().cpu() for k, v in net.rnn.state_dict().items()})
    fc = torch.nn.Linear(20, V).double()
    fc.load_state_dict({k: v.double().cpu() for k, v in net.fc.state_dict().items()})
    w64, c64 = [u.detach().double().cpu().requires_grad_() for u in (words, code)]
    z = fc(rnn(torch.cat((w64, c64[:, None].expand(B, T, Z)), 2))[0].reshape(B * T, 20))
    lp = torch.log_softmax(z, 1).gather(1, t.cpu()[:, None])[:, 0]
    old = (lp.detach() - shift.double().cpu()).float()
    wd = w.double().cpu().view(-1)
    if form == "policy":
        rho, Ad = (lp - old.double()).exp(), A.double().cpu()
        want = -(wd * torch.minimum(rho * Ad, rho.clamp(0.8, 1.2) * Ad)).sum()
    else:
        gain = (wd * lp).view(B, T).sum(1) - sref.double().cpu()
        want = -torch.nn.functional.logsigmoid(0.1 * (gain[:B // 2] - gain[B // 2:])).mean()
    want.backward()

    logits, _ = net(words, code, 0.0)
    logits = logits.view(B * T, V)
    if form == "policy":
        loss = hnn.policy_loss(logits, t, A, w.view(-1), old_logp=old.to(dev))[0]
    else:
        loss = hnn.preference_loss(logits, t, w, sref, beta=0.1)[0]
    loss.backward()
    # norms: 2 layers of 7 steps there and back, 8 u a step, and 64 u for the projection and the loss: below 300 u
    assert abs(float(loss.detach()) - float(want.detach())) <= 300 * U * float((wd * lp.detach().abs()).sum())
    pairs = list(zip(net.rnn.flat_weights(), [getattr(rnn, k + "_l%d" % l) for l in (0, 1) for k in
                                              ("weight_ih", "weight_hh", "bias_ih", "bias_hh")]))
    pairs += [(net.fc.weight, fc.weight), (net.fc.bias, fc.bias), (words, w64), (code, c64)]
    for k, (a, b) in enumerate(pairs):
        assert (a.grad.double().cpu() - b.grad).norm() <= 300 * U * b.grad.norm(), k


def test_other_streams(dev):
    """Every operator on a side stream, two at once, against the default stream's answers."""
    M, V = 64, 5000
    jobs = []
    for k in range(2):
        x, t, A, w, old, ref = make_policy(M, V, BF16 if k else F32, 70 + k, dev)
        h = torch.randn(500, 300, device=dev, generator=gen(k)).to(x.dtype)
        jobs.append((x, t, A, w, old, ref, h))

    def work(x, t, A, w, old, ref, h):
        d = torch.empty_like(x)
        loss, logp = ops.policy_loss(x, t, A, w, old_logp=old, ref_logp=ref, kl_coef=0.1, dlogits=d)
        pl, pm, ps = ops.preference_loss(x, t, w.view(8, 8), torch.zeros(8, device=dev), beta=0.1)
        y, mean, rstd = ops.layer_norm_fwd(h)
        dx, _, db = ops.layer_norm_bwd(h, h, None, mean, rstd)
        out = [torch.empty_like(d), torch.empty_like(dx)]
        n = ops.clip_grad_norm([d, dx], 0.5, out=out)
        return [loss, logp, d, pl, pm, ps, y, dx, db, n] + out

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(*j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured(dev):
    """The whole chain of kernels in one graph, replayed on changing inputs with eager work in between; two graphs captured
    on one stream and replayed at once on two do not share scratch memory."""
    M, V, H = 48, 3001, 300

    def fresh(seed):
        x, t, A, w, old, ref = make_policy(M, V, F32, seed, dev)
        return [x, t, A, w, old, ref, torch.randn(M, H, device=dev, generator=gen(seed))]

    def work(x, t, A, w, old, ref, h):
        d = torch.empty_like(x)
        loss, logp = ops.policy_loss(x, t, A, w, old_logp=old, ref_logp=ref, kl_coef=0.1, dlogits=d)
        d2 = torch.empty_like(x)
        pl, pm, ps = ops.preference_loss(x, t, w.view(6, 8), logp[:6].contiguous(), beta=0.1, dlogits=d2)
        y, mean, rstd = ops.layer_norm_fwd(h)
        dx, _, db = ops.layer_norm_bwd(y, h, None, mean, rstd)
        n = ops.clip_grad_norm([d, d2, dx], 0.5)
        return [loss, logp, d, d2, pl, pm, ps, y, dx, db, n]

    side = torch.cuda.Stream()
    sets = []
    with torch.cuda.stream(side):
        work(*fresh(1))
        torch.cuda.synchronize()
        for k in range(2):
            ins = fresh(10 + k)
            graph = torch.cuda.CUDAGraph()
            with ops.capture_without_gc():
                with torch.cuda.graph(graph, stream=side):
                    outs = work(*ins)
            sets.append((graph, ins, outs))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        news = [fresh(100 + 10 * rep + k) for k in range(2)]
        wants = [work(*n) for n in news]
        for (graph, ins, _), n in zip(sets, news):
            for a, b in zip(ins, n):
                a.copy_(b)
        torch.cuda.synchronize()
        for s, (graph, _, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs), want in zip(sets, wants):
            assert all(torch.equal(p, q) for p, q in zip(outs, want)), rep


def test_captured_modules(dev):
    """Forward and backward of the differentiable forms in a graph, replayed on changing inputs; a capture over parameters
    that a graph built outside of it still holds is refused before anything of it is recorded."""
    M, H = 24, 300
    ln = hnn.LayerNorm(H).to(dev)
    t = torch.randint(0, H, (M,), device=dev, generator=gen(1))
    A, w = torch.randn(M, device=dev, generator=gen(2)), torch.rand(M, device=dev, generator=gen(3))
    x = torch.randn(M, H, device=dev, generator=gen(4))

    def step(v):
        loss, _ = hnn.policy_loss(ln(v), t, A, w)
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        alive = ln(x)  # an eager graph over the same parameters
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(graph, stream=side):
                ln(x)
        with torch.no_grad():  # no backward pass can follow: taken
            free = torch.cuda.CUDAGraph()
            with ops.capture_without_gc():
                with torch.cuda.graph(free, stream=side):
                    y = ln(x)
            free.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, alive)
        del alive
        torch.cuda.synchronize()
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with ops.capture_without_gc():
            with torch.cuda.graph(graph, stream=side):
                out = step(static)
    torch.cuda.synchronize()
    grads = [ln.weight.grad, ln.bias.grad]
    for rep in range(4):
        new = torch.randn(M, H, device=dev, generator=gen(20 + rep))
        twin = hnn.LayerNorm(H).to(dev)  # the eager answer, on parameters of its own
        loss, _ = hnn.policy_loss(twin(new), t, A, w)
        loss.backward()
        static.copy_(new)
        for gr in grads:
            gr.zero_()  # (the captured accumulation adds where it did not create)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, loss.detach())
        assert torch.equal(grads[0], twin.weight.grad) and torch.equal(grads[1], twin.bias.grad)


def small_engine(dev, **kw):
    from ldrs_amd.model.cgn import Controlled_Generation_Sentence
    from ldrs_amd.utils.config import Config
    from oracle import cgn_oracle as O
    dims = dict(word_embed_size=12, kernels=((1, 3), (2, 5), (3, 4)), encoder_rnn_size=16, latent_variable_size=6,
                decoder_rnn_size=20, sentiment_kernel_size=(3, 4, 5), sentiment_kernel_num=6)
    ocfg = O.OracleConfig(max_word_len=7, max_seq_len=5, word_vocab_size=50, char_vocab_size=20, **dims)
    torch.manual_seed(2)
    model = Controlled_Generation_Sentence(Config(7, 5, 50, 20, 1e-3, 7.9, 0.1, 0.1, 1.0, **dims, **kw),
                                           O.synthetic_word_embed(ocfg)).to(dev)
    eng = model.step_engine()
    data = {k: v.to(dev).contiguous() for k, v in O.synthetic_batch(ocfg, 4, 5, seed=1).items()}
    return model, eng, {g: eng.new_optimizer(g) for g in ("disc", "enc", "gen")}, data


def test_training_step_is_clipped(dev):
    """Config(max_grad_norm=...): the wake-sleep step clips every optimizer group, eager and replayed from a graph."""
    from ldrs_amd.hip.graph import GraphedWakeSleep
    plain, wide, tight = small_engine(dev), small_engine(dev, max_grad_norm=1e6), small_engine(dev, max_grad_norm=0.01)
    for _, eng, opts, data in (plain, wide, tight):
        eng.wake_sleep(opts, data, 0.5, 0.9)
    for (n, p), (_, q) in zip(plain[0].named_parameters(), wide[0].named_parameters()):
        assert torch.equal(p, q), n  # a bound that nothing reaches changes no bit
    for g in ("disc", "enc", "gen"):
        grads = [t for t in tight[1].arenas[g].grads.values()]
        want = norm64(grads)
        assert want > 0.01 and abs(float(tight[1].grad_norms[g]) - want) <= 2 * U * want
        # first step: m = (1 - beta1) * clipped gradient
        m = float(tight[2][g].m.double().norm())
        assert abs(m - 0.1 * 0.01) <= 1e-6 * 0.1 * 0.01 + 0.1 * 0.01 * 1e-6 / want
    assert not plain[1].grad_norms
    eager, graphed = small_engine(dev, max_grad_norm=0.01), small_engine(dev, max_grad_norm=0.01)
    for _ in range(4):
        eager[1].wake_sleep(eager[2], eager[3], 0.5, 0.9)
    rep = GraphedWakeSleep(graphed[1], graphed[2], graphed[3], warmup_kld=0.5, warmup_tau=0.9)
    for _ in range(3):
        rep(0.5, 0.9, graphed[3])
        torch.cuda.synchronize()
    for (n, p), (_, q) in zip(eager[0].named_parameters(), graphed[0].named_parameters()):
        err = (p - q).abs().max().item() / max(p.abs().max().item(), 1e-12)
        assert err <= 2e-6, (n, err)  # (the bias corrections are formed on the device there)
    with pytest.raises(ValueError):
        small_engine(dev, max_grad_norm=-1.0)
