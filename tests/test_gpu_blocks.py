"""The RMS norm, the gated linear layer and gradient clipping against plain computations in 64 bits.

Tolerances are sums of what each rounding can do: half a step of the output's type relative to its value
(U[t]), the same for each operand that is stored in between, and fp32 arithmetic at 2^-24 a step (2^-23
where the matrix unit accumulates: its steps may truncate) times the number of steps and the sum of
the absolute terms."""
import math

import pytest
import torch

from pointcloud_style_transfer_amd import _hip
from pointcloud_style_transfer_amd.models import (GatedLinear, RMSNorm, gated_linear, gated_linear_quant, quant_rows,
                                                  rms_norm, rms_norm_quant)
from pointcloud_style_transfer_amd.utils import clip_grad_norm_, clip_grads

pytestmark = pytest.mark.gpu

F32, BF, F16, E4 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF, F16)}
TINY = {F32: 2.0 ** -149, BF: 2.0 ** -133, F16: 2.0 ** -24}  # a step of the subnormals
R = 2.0 ** -24


def rand(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def within(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs() - bound
    assert bool(torch.isfinite(got.float()).all()), what
    worst = float(off.detach().max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: over the bound by {worst:.3g} (|want| there {float(want.flatten()[off.argmax()].abs()):.3g})"


# ------------------------------------------------------------------------------------------ norm
def norm_ref(x, w, r, eps):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    sd = s.double()
    rho = 1 / (sd.square().mean(-1, keepdim=True) + eps).sqrt()
    return s, sd * rho, rho, sd * rho * w.double()


# a thread adds at most 32 squares, then 6 exchanges and 8 waves; all terms positive: relative 2^-24 each,
# half of it on the root, and a few operations of one rounding
NORM_REL = 28 * R


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 7), (17, 64), (5, 129), (33, 256), (2, 511), (9, 1000), (4, 2048), (3, 2049),
                                 (2, 5001), (1, 8192), (2, 16384)])
@pytest.mark.parametrize("res", [False, True])
def test_norm_forward(M, D, dtype, res):
    x, w = rand(1, M, D, dtype=dtype), rand(2, D, dtype=dtype if D % 2 else F32) + 1
    r = rand(3, M, D, dtype=dtype, scale=2) if res else None
    s, n, rho, y = norm_ref(x, w, r, 1e-6)
    with torch.no_grad():
        got = rms_norm(x, w, r)
    if res:
        got, gs = got
        assert torch.equal(gs, s)
    within(got, y, (U[dtype] + NORM_REL) * y.abs() + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("M,D,res", [(1, 5, True), (37, 64, False), (1030, 256, True), (5000, 100, False), (77, 1000, True),
                                     (40, 2049, True), (6, 8191, False), (3, 16384, True), (700, 300, True)])
def test_norm_backward(M, D, dtype, res):
    x, w = rand(1, M, D, dtype=dtype), rand(2, D, dtype=dtype if D % 2 else F32) + 1
    r = rand(3, M, D, dtype=dtype) if res else None
    dy, ds = rand(4, M, D, dtype=dtype), rand(5, M, D, dtype=dtype) if res else None
    leaves = [t.requires_grad_() for t in ([x, w] if r is None else [x, w, r])]
    out = rms_norm(x, w, r)
    grads = torch.autograd.grad(out, leaves, dy if r is None else (dy, ds))
    s, n, rho, _ = norm_ref(x.detach(), w.detach(), None if r is None else r.detach(), 1e-6)
    a = dy.double() * w.detach().double()
    mean = (a * n).mean(-1, keepdim=True)
    dx = rho * (a - n * mean)
    size = rho * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True))
    if res:
        dx, size = dx + ds.double(), size + ds.double().abs()
        assert torch.equal(grads[0], grads[2])
    # n carries NORM_REL, the row sum 46 steps, the rest a few: 128 steps of the absolute terms
    within(grads[0], dx, U[dtype] * dx.abs() + 128 * R * size + TINY[dtype], "dx")
    terms = (dy.double() * n).abs().sum(0)
    rows = math.ceil(M / 512) + 16  # rows a thread adds in fp32, and the work-group's
    dw = (dy.double() * n).sum(0)
    within(grads[1], dw, U[w.dtype] * dw.abs() + (rows + 32) * R * terms + TINY[w.dtype], "dw")


def test_norm_against_differences():
    x, w, r = (rand(i, 4, 24).double() for i in (1, 2, 3))
    w = w[0]
    dy, ds = rand(4, 4, 24), rand(5, 4, 24)

    def f(x, w, r):
        s = x + r
        y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        return float((y * dy.double()).sum() + (s * ds.double()).sum())

    leaves = [t.float().requires_grad_() for t in (x, w, r)]
    grads = torch.autograd.grad(rms_norm(*leaves), leaves, (dy, ds))
    h = 1e-5
    for k, (t, g) in enumerate(zip((x, w, r), grads)):
        for at in (0, 5, t.numel() - 1):
            args = [v.clone() for v in (x, w, r)]
            args[k].view(-1)[at] += h
            up = f(*args)
            args[k].view(-1)[at] -= 2 * h
            d = (up - f(*args)) / (2 * h)
            # differences: h^2 of a third derivative of order 10, and 1e-12 / h of cancellation; fp32: 1e-5
            assert abs(d - float(g.view(-1)[at])) < 2e-5 * max(1.0, abs(d))


def test_norm_only_the_stream_goes_on():
    x, w, r = rand(1, 8, 64).requires_grad_(), rand(2, 64).requires_grad_(), rand(3, 8, 64).requires_grad_()
    ds = rand(4, 8, 64)
    y, s = rms_norm(x, w, r)
    gx, gw, gr = torch.autograd.grad(s, [x, w, r], ds, allow_unused=True)
    assert torch.equal(gx, ds) and torch.equal(gr, ds) and gw is None
    y, s = rms_norm(x, w, r)
    g1 = torch.autograd.grad(y, [x, w, r], ds)
    g2 = torch.autograd.grad(rms_norm(x, w, r), [x, w, r], (ds, torch.zeros_like(ds)))
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("M,D,res", [(1, 1, False), (5, 8, True), (33, 256, True), (7, 1001, True), (3, 4096, False), (2, 16384, True)])
def test_norm_quant(M, D, dtype, res):
    x, w = rand(1, M, D, dtype=dtype), rand(2, D, dtype=F32) + 1
    r = rand(3, M, D, dtype=dtype) if res else None
    x[0] = 0
    if res:
        r[0] = 0
    got = rms_norm_quant(x, w, r)
    s, _, _, y = norm_ref(x, w, r, 1e-6)
    if res:
        assert torch.equal(got[2], s)
    q, sc = got[0].double(), got[1].double()
    want = y.abs().amax(-1) / 448
    want = torch.where(want == 0, torch.ones_like(want), want)
    within(got[1], want, (NORM_REL + 2 * R) * want, "scale")
    assert float(sc[0]) == 1.0 and not bool(q[0].any())
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the smallest normal value
    within((q * sc[:, None]), y, 2.0 ** -4 * y.abs() + 2.0 ** -10 * sc[:, None] + (NORM_REL + 4 * R) * y.abs(), "q")
    if M > 1 or not res:
        assert float(q.abs().amax()) in (0.0, 448.0)


def test_quant_rows_and_nonfinite():
    x = rand(1, 6, 200, dtype=BF, scale=3)
    q, sc = quant_rows(x)
    # (a division by a Python scalar multiplies by its rounded reciprocal: divide in 64 bits, round once)
    assert torch.equal(sc, (x.double().abs().amax(-1) / 448).float())
    assert torch.equal(q.float(), (x.float() / sc[:, None]).to(E4).float())
    x[1, 3], x[2, 4] = math.nan, math.inf
    q, sc = quant_rows(x)
    assert math.isnan(float(q[1].float()[3])) and int(torch.isnan(q[1].float()).sum()) == 1
    assert math.isinf(float(sc[2]))
    y = rms_norm(x, torch.ones(200, device="cuda", dtype=BF))
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[3:]).all())


def test_norm_no_rows_and_strides():
    w = (rand(2, 64) + 1).requires_grad_()
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(rms_norm(x, w), [x, w], torch.empty(0, 64, device="cuda"))
    assert gx.shape == (0, 64) and not bool(gw.any())
    big = rand(3, 4, 9, 130, dtype=BF)
    v = big[:, 1:8:2, 1:65]  # odd offset, steps between rows
    y, s = rms_norm(v, w.detach().to(BF), v)
    yc, sc = rms_norm(v.contiguous(), w.detach().to(BF), v.contiguous())
    assert torch.equal(y, yc) and torch.equal(s, sc)
    flat = rand(4, 65 * 7 + 1, dtype=BF)[1:].view(7, 65)  # rows start off 16-byte boundaries
    w65 = (rand(5, 66, dtype=BF) + 1)[1:]
    assert torch.equal(rms_norm(flat, w65), rms_norm(flat.clone(), w65.clone()))
    t = v.transpose(0, 1)
    assert torch.equal(rms_norm(t, w.detach().to(BF)), rms_norm(t.contiguous(), w.detach().to(BF)))


def test_norm_past_31_bits():
    M, D = 140000, 16384  # 2.29e9 values
    x = torch.empty(M, D, device="cuda", dtype=BF)
    x[:8] = rand(1, 8, D, dtype=BF)
    x[-8:] = rand(2, 8, D, dtype=BF)
    w = torch.ones(D, device="cuda", dtype=BF)
    y, _, rho = _hip.rms_norm(x, w, stats=True)
    for part in (slice(0, 8), slice(M - 8, M)):
        assert torch.equal(y[part], _hip.rms_norm(x[part].clone(), w)[0])
    dx, dw = _hip.rms_norm_bwd(x, w, rho, y, need_dw=False)
    assert torch.equal(dx[-8:], _hip.rms_norm_bwd(x[-8:].clone(), w, rho[-8:].clone(), y[-8:].clone(), need_dw=False)[0])


# ------------------------------------------------------------------------------------------ gated
def act_ref(g, act):
    if act == "silu":
        e = torch.sigmoid(g)
        return g * e, e * (1 + g * (1 - e))
    if act == "gelu":
        c = torch.special.ndtr(g)
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).double()


def gated_ref(x, wg, wu, bg, bu, act):
    """g, u and what fp32 accumulation over D terms may be off."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = x.abs() @ wg.t().abs(), x.abs() @ wu.t().abs()
    if bg is not None:
        g, u, eg, eu = g + bg.double(), u + bu.double(), eg + bg.double().abs(), eu + bu.double().abs()
    steps = (x.shape[1] + 8) * 2.0 ** -23
    return g, u, steps * eg, steps * eu


# the activation's own error in fp32: a dozen roundings of |act| <= |g| and of derivatives <= 1.13
ACT_REL = 16 * R


def check_h(h, g, u, eg, eu, act, dtype):
    a, _ = act_ref(g, act)
    want = a * u
    b = 1.13 * eg * (u.abs() + eu) + a.abs() * eu + ACT_REL * g.abs() * u.abs()
    within(h, want, U[dtype] * (want.abs() + b) + b + TINY[dtype], "h")


SHAPES = [(1, 1, 1), (1, 64, 64), (3, 8, 5), (2, 7, 3), (17, 33, 70), (64, 64, 64), (127, 100, 65), (128, 256, 128),
          (130, 257, 129), (129, 72, 200), (300, 520, 130), (1, 1000, 333), (5, 2048, 96), (16, 513, 40), (31, 96, 50),
          (33, 1024, 48), (63, 515, 17), (65, 515, 17)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,D,F", SHAPES)
def test_gated_forward(M, D, F, dtype):
    act = ["silu", "gelu", "relu"][(M + F) % 3]
    x, k = rand(1, M, D, dtype=dtype), D ** -0.5
    wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
    bias = (M + D) % 2 == 0
    bg, bu = (rand(4, F, dtype=dtype), rand(5, F, dtype=dtype)) if bias else (None, None)
    h = gated_linear(x, wg, wu, bg, bu, act)
    check_h(h, *gated_ref(x, wg, wu, bg, bu, act), act, dtype)


def check_grads(x, wg, wu, bg, bu, act, dh, grads, dtype, wdtype=None):
    """grads: dx, dwg, dwu, dbg, dbu of gated_linear; dg and du are stored in dtype in between."""
    wdtype = wdtype or dtype
    g, u, eg, eu = gated_ref(x, wg, wu, bg, bu, act)
    a, da = act_ref(g, act)
    dh = dh.double()
    dg, du = dh * u * da, dh * a
    curve = torch.full_like(g, 1.0)  # |act''| <= 0.8 for silu and gelu
    if act == "relu":
        curve = torch.where(g.abs() <= eg, 1 / eg.clamp(min=1e-300), torch.zeros_like(g))  # may fall on either side
    bdg = dh.abs() * (eu * 1.13 + (u.abs() + eu) * (curve * eg).clamp(max=1.13) + ACT_REL * (u.abs() + eu) * (1 + g.abs()))
    bdu = dh.abs() * (1.13 * eg + ACT_REL * g.abs())
    edg, edu = bdg + U[dtype] * (dg.abs() + bdg) + TINY[dtype], bdu + U[dtype] * (du.abs() + bdu) + TINY[dtype]
    xd, wgd, wud = x.double().abs(), wg.double().abs(), wu.double().abs()

    def product(want, a, ea, b, k, t, what, got):
        if got is None:
            return
        size = (a.abs() + ea) @ b
        e = ea @ b + (k + 8) * 2.0 ** -23 * size
        within(got, want, e + U[t] * (want.abs() + e) + TINY[t], what)

    F = wg.shape[0]
    product(dg @ wg.double() + du @ wu.double(), torch.cat([dg, du], 1), torch.cat([edg, edu], 1), torch.cat([wgd, wud]),
            2 * F + 128, dtype, "dx", grads[0])
    M = x.shape[0]
    product(dg.t() @ x.double(), dg.t(), edg.t(), xd, M + 256, wdtype, "dw_gate", grads[1])
    product(du.t() @ x.double(), du.t(), edu.t(), xd, M + 256, wdtype, "dw_up", grads[2])
    for d, b, got, what in ((dg, bdg, grads[3], "db_gate"), (du, bdu, grads[4], "db_up")):
        if got is not None:
            want, e = d.sum(0), b.sum(0) + 80 * R * d.abs().sum(0)  # 4 rows a lane, 16 lanes; then fp64
            within(got, want, e + U[got.dtype] * (want.abs() + e) + TINY[got.dtype], what)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,D,F", SHAPES + [(1000, 64, 96), (2100, 130, 40), (4097, 48, 33)])
def test_gated_backward(M, D, F, dtype):
    act = ["silu", "gelu", "relu"][(M + F) % 3]
    x, k = rand(1, M, D, dtype=dtype), D ** -0.5
    wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
    bias = (M + D) % 2 == 0
    bt = F32 if F % 2 else dtype
    bg, bu = (rand(4, F, dtype=bt), rand(5, F, dtype=bt)) if bias else (None, None)
    dh = rand(6, M, F, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    h = gated_linear(x, wg, wu, bg, bu, act)
    grads = list(torch.autograd.grad(h, leaves, dh)) + ([] if bias else [None, None])
    det = [None if t is None else t.detach() for t in (x, wg, wu, bg, bu)]
    check_grads(*det, act, dh, grads, dtype)


def test_gated_large_tiles():
    """Sizes that take the large tiles in every product, with rows, columns and k that end inside one."""
    for M, D, F, dtype in ((6500, 1104, 1100, BF), (5200, 2311, 2570, F16), (5200, 2312, 2571, BF), (5200, 2310, 2561, F32)):
        x, k = rand(1, M, D, dtype=dtype), D ** -0.5
        wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
        dh = rand(6, M, F, dtype=dtype)
        check_h(_hip.gated_linear(x, wg, wu), *gated_ref(x, wg, wu, None, None, "silu"), "silu", dtype)
        check_grads(x, wg, wu, None, None, "silu", dh, _hip.gated_linear_bwd(x, wg, wu, dh), dtype)


# many rows of few columns (the weights stay in LDS), rows, columns and k that end inside a tile
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M,D,F", [(9000, 130, 999), (30000, 200, 301), (20011, 72, 701), (24577, 128, 640), (20000, 256, 512),
                                   (40001, 33, 1000), (17000, 255, 385)])
def test_gated_narrow(M, D, F, dtype):
    act, bt = ["silu", "gelu", "relu"][F % 3], F32 if D % 2 else dtype
    x, k = rand(1, M, D, dtype=dtype), D ** -0.5
    wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
    for bg, bu in ((rand(4, F, dtype=bt), rand(5, F, dtype=bt)), (None, None)):
        h = _hip.gated_linear(x, wg, wu, bg, bu, act)
        check_h(h, *gated_ref(x, wg, wu, bg, bu, act), act, dtype)
    # a row's value does not depend on the rows beside it, whichever wave takes it
    keep = [0, 31, 32, 63, 64, 4095, M - 2, M - 1]
    y = torch.zeros_like(x)
    y[keep] = x[keep]
    assert torch.equal(_hip.gated_linear(y, wg, wu, act=act)[keep], h[keep])
    shifted = torch.empty(x.numel() + 1, device="cuda", dtype=dtype)[1:].view_as(x).copy_(x)
    assert torch.equal(_hip.gated_linear(shifted, wg, wu, act=act), h)
    y = x.clone()
    y[5] = math.inf
    other = _hip.gated_linear(y, wg, wu, act=act)
    assert torch.equal(other[6:], h[6:]) and torch.equal(other[:5], h[:5])


# 1 to 128 rows on either kernel, rows of every alignment, the last piece of a row of any length
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,D,F", [(1, 1, 3), (2, 3, 17), (17, 7, 16), (66, 31, 40), (100, 519, 130), (128, 1000, 64), (128, 4096, 48),
                                   (97, 130, 300), (127, 2050, 33), (65, 64, 8)])
def test_gated_few_rows(M, D, F, dtype):
    act = ["silu", "gelu", "relu"][M % 3]
    k = D ** -0.5
    bx = torch.full((M * D + 40,), math.nan, device="cuda", dtype=dtype)
    bw = torch.full((2 * F * D + 40,), math.nan, device="cuda", dtype=dtype)
    for at in (0, 1, 8):  # elements in front; what lies around the operands is NaN
        x, wg, wu = bx[at:at + M * D].view(M, D), bw[at:at + F * D].view(F, D), bw[at + F * D:at + 2 * F * D].view(F, D)
        x.copy_(rand(1, M, D))
        wg.copy_(rand(2, F, D, scale=k))
        wu.copy_(rand(3, F, D, scale=k))
        b = rand(4, F)
        check_h(_hip.gated_linear(x, wg, wu, b, b, act), *gated_ref(x, wg, wu, b, b, act), act, dtype)
        if dtype == BF:
            (q, xs), (g8, gs), (u8, us) = quant_rows(x), quant_rows(wg), quant_rows(wu)
            h = gated_linear_quant(q, xs, g8, gs, u8, us, b, b, act=act)
            full = [torch.cat([t.view(torch.uint8), t.view(torch.uint8)[:1]]).view(torch.float8_e4m3fn)[:n] for t, n in ((q, M), (g8, F), (u8, F))]
            assert torch.equal(h, gated_linear_quant(full[0], xs, full[1], gs, full[2], us, b, b, act=act))
        bx.fill_(math.nan)
        bw.fill_(math.nan)


# the backward of many rows of 129 to 256 columns (the weights stay in LDS): rows and columns that end inside a tile,
# odd sizes, column sums of each wave's rows
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M,D,F", [(60000, 200, 301), (60001, 200, 300), (61441, 130, 640), (60001, 256, 512), (50000, 255, 385), (40000, 136, 1000)])
def test_gated_narrow_backward(M, D, F, dtype):
    act, bt = ["silu", "gelu", "relu"][F % 3], F32 if D % 4 else dtype
    x, k = rand(1, M, D, dtype=dtype), D ** -0.5
    wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
    dh, bg, bu = rand(6, M, F, dtype=dtype), rand(4, F, dtype=bt), rand(5, F, dtype=bt)
    grads = _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, act)
    check_grads(x, wg, wu, bg, bu, act, dh, grads, dtype)
    for a, b in zip(grads, _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, act)):
        assert torch.equal(a, b)
    shifted = torch.empty(dh.numel() + 1, device="cuda", dtype=dtype)[1:].view_as(dh).copy_(dh)
    for a, b in zip(grads[:3], _hip.gated_linear_bwd(x, wg, wu, shifted, bg, bu, act)):
        assert torch.equal(a, b)
    bare = _hip.gated_linear_bwd(x, wg, wu, dh, act=act)
    check_grads(x, wg, wu, None, None, act, dh, bare, dtype)


# few tiles and a long k, which is split: in h (long D), in dx (long F), in dW (many rows)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,D,F", [(65, 4000, 70), (100, 2999, 301), (300, 2000, 40), (70, 1000, 33), (5000, 65, 701),
                                   (9000, 64, 1000), (700, 520, 200), (2000, 1030, 72),
                                   (33, 4100, 5200)])
def test_gated_splits(M, D, F, dtype):
    act = ["silu", "gelu", "relu"][M % 3]
    x, k = rand(1, M, D, dtype=dtype), D ** -0.5
    wg, wu = rand(2, F, D, dtype=dtype, scale=k), rand(3, F, D, dtype=dtype, scale=k)
    bt = F32 if F % 2 else dtype
    bg, bu, dh = rand(4, F, dtype=bt), rand(5, F, dtype=bt), rand(6, M, F, dtype=dtype)
    h = _hip.gated_linear(x, wg, wu, bg, bu, act)
    check_h(h, *gated_ref(x, wg, wu, bg, bu, act), act, dtype)
    grads = _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, act)
    check_grads(x, wg, wu, bg, bu, act, dh, grads, dtype)
    for a, b in zip(grads, _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, act)):
        assert torch.equal(a, b)
    assert torch.equal(h, _hip.gated_linear(x, wg, wu, bg, bu, act))
    need = (1, 0, 0, 0, 1)
    for n, a, b in zip(need, grads, _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, act, need=need)):
        assert torch.equal(a, b) if n else b is None


def test_gated_against_differences():
    M, D, F = 3, 9, 7
    x, wg, wu, bg, bu = rand(1, M, D), rand(2, F, D), rand(3, F, D), rand(4, F), rand(5, F)
    dh = rand(6, M, F)
    for act in ("silu", "gelu"):
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
        grads = torch.autograd.grad(gated_linear(*leaves, act=act), leaves, dh)

        def f(args):
            g, u, _, _ = gated_ref(*args, act)
            return float((act_ref(g, act)[0] * u * dh.double()).sum())

        for k in range(5):
            for at in (0, leaves[k].numel() - 1):
                args = [t.double() for t in (x, wg, wu, bg, bu)]
                args[k] = args[k].clone()
                args[k].view(-1)[at] += 1e-5
                up = f(args)
                args[k].view(-1)[at] -= 2e-5
                d = (up - f(args)) / 2e-5
                assert abs(d - float(grads[k].view(-1)[at])) < 1e-4 * max(1.0, abs(d))


@pytest.mark.parametrize("need", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 1), (0, 0, 0, 1, 0), (1, 1, 1, 1, 1)])
def test_gated_needed_gradients(need):
    x, wg, wu, bg, bu = rand(1, 70, 40, dtype=BF), rand(2, 50, 40, dtype=BF), rand(3, 50, 40, dtype=BF), rand(4, 50), rand(5, 50)
    dh = rand(6, 70, 50, dtype=BF)
    every = _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu)
    some = _hip.gated_linear_bwd(x, wg, wu, dh, bg, bu, need=need)
    for n, a, b in zip(need, some, every):
        assert (a is None) if not n else torch.equal(a, b)


@pytest.mark.parametrize("out", [BF, F16])
@pytest.mark.parametrize("M,D,F,bias", [(1, 16, 16, True), (3, 5, 7, False), (65, 130, 70, True), (200, 256, 300, False),
                                        (140, 1000, 129, True), (6500, 256, 1100, False), (70, 4000, 40, True),
                                        (300, 2050, 65, False)])
def test_gated_quant(M, D, F, bias, out):
    x, k = rand(1, M, D, dtype=BF), D ** -0.5
    q, xs = rms_norm_quant(x, torch.ones(D, device="cuda"))
    (wg, gs), (wu, us) = quant_rows(rand(2, F, D, scale=k)), quant_rows(rand(3, F, D, scale=k))
    bg, bu = (rand(4, F), rand(5, F)) if bias else (None, None)
    h = gated_linear_quant(q, xs, wg, gs, wu, us, bg, bu, act="gelu", out_dtype=out)
    deq = lambda v, s: v.double() * s.double()[:, None]  # noqa: E731
    xd, wgd, wud = deq(q, xs), deq(wg, gs), deq(wu, us)
    g, u, eg, eu = gated_ref(xd, wgd, wud, bg, bu, "gelu")

    def group_sums(x, w):
        """The matrix unit adds the e4m3 products of 8 consecutive k at 14 bits below the binade of their
        largest (measured: 2^17 + 2^3 is kept, 2^2 is not), so each of the 7 others loses less than 2^-14 of it."""
        pad = (-x.shape[1]) % 8
        x, w = (torch.nn.functional.pad(t.abs(), (0, pad)) for t in (x, w))
        top = torch.zeros(x.shape[0], w.shape[0], device="cuda", dtype=torch.float64)
        for k in range(0, x.shape[1], 8):
            top += (x[:, None, k:k + 8] * w[None, :, k:k + 8]).amax(-1) if x.shape[0] < 1000 else \
                x[:, k:k + 8].amax(-1)[:, None] * w[:, k:k + 8].amax(-1)[None]
        return 7 * 2.0 ** -14 * top

    check_h(h, g, u, eg + group_sums(xd, wgd), eu + group_sums(xd, wud), "gelu", out)
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        gated_linear_quant(q, xs, wg, gs, wu, us, bg, bu, out_dtype=F32)


def test_gated_special_values():
    x, wg, wu = rand(1, 40, 64, dtype=BF), rand(2, 48, 64, dtype=BF), rand(3, 48, 64, dtype=BF)
    x[3, 5] = math.nan
    x[7] = 1e30
    x[9] = 0
    for act in ("silu", "gelu", "relu"):
        h = gated_linear(x, wg, wu, act=act)
        assert bool(torch.isnan(h[3]).all()) and not bool(h[9].any())
        rest = [i for i in range(40) if i not in (3, 7)]
        assert bool(torch.isfinite(h[rest]).all())
        clean = x.clone()
        clean[3] = clean[7] = 0
        assert torch.equal(h[rest], gated_linear(clean, wg, wu, act=act)[rest])
    # NaN behind the operands' ends does not leak in: rows and columns of larger buffers
    bx = torch.full((200, 72), math.nan, device="cuda", dtype=BF)
    bw = torch.full((200, 72), math.nan, device="cuda", dtype=BF)
    bx[:33, :70], bw[:37, :70] = rand(4, 33, 70, dtype=BF), rand(5, 37, 70, dtype=BF)
    xv, wv = bx[:33, :70], bw[:37, :70]
    assert torch.equal(gated_linear(xv, wv, wv), gated_linear(xv.contiguous(), wv.contiguous(), wv.contiguous()))
    bx[:33, 70:] = 0
    full = torch.cat([bx[:33], bx[100:]])
    got = gated_linear(full, bx[:33].clone(), bx[:33].clone())[:33]
    assert torch.equal(got, gated_linear(bx[:33], bx[:33], bx[:33]))


def test_gated_alignment_and_strides():
    x, wg, wu = rand(1, 50, 64, dtype=F16), rand(2, 40, 64, dtype=F16), rand(3, 40, 64, dtype=F16)
    dh = rand(4, 50, 40, dtype=F16)
    want, grads = _hip.gated_linear(x, wg, wu), _hip.gated_linear_bwd(x, wg, wu, dh)

    def shifted(t):
        b = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view_as(t)
        return b.copy_(t)

    for a in ((shifted(x), wg, wu), (x, shifted(wg), wu), (x, wg, shifted(wu)), (x.t().contiguous().t(), wg, wu.t().contiguous().t())):
        assert torch.equal(_hip.gated_linear(*a), want)
        for u, v in zip(_hip.gated_linear_bwd(*a, shifted(dh)), grads):
            assert (u is None and v is None) or torch.equal(u, v)
    y = gated_linear(x.view(5, 10, 64), wg, wu)
    assert torch.equal(y.view(50, 40), want)
    assert gated_linear(x[:0], wg, wu).shape == (0, 40)
    e = [t.clone().requires_grad_() for t in (x[:0], wg, wu)]
    g = torch.autograd.grad(gated_linear(*e), e, torch.empty(0, 40, device="cuda", dtype=F16))
    assert g[0].shape == (0, 64) and not bool(g[1].any()) and not bool(g[2].any())


def test_gated_past_31_bits():
    M, D, F = 70016, 64, 32768  # h of 2.29e9 values
    x, wg, wu = rand(1, M, D, dtype=BF), rand(2, F, D, dtype=BF), rand(3, F, D, dtype=BF)
    h = _hip.gated_linear(x, wg, wu)
    for part in (slice(0, 40), slice(M - 40, M)):
        check_h(h[part], *gated_ref(x[part], wg, wu, None, None, "silu"), "silu", BF)
    dx = _hip.gated_linear_bwd(x, wg, wu, h, need=(1, 0, 0, 0, 0))[0]
    tail = _hip.gated_linear_bwd(x[-40:].clone(), wg, wu, h[-40:].clone(), need=(1, 0, 0, 0, 0))[0]
    # another tile shape may add dx's terms in another order: 2 F terms of fp32, both sides
    size = (2 * F + 136) * 2.0 ** -23 * tail.double().abs().mean() * 64
    assert float((dx[-40:].double() - tail.double()).abs().max()) <= float(2 * U[BF] * tail.double().abs().max() + size)


def test_gated_autocast():
    x, wg, wu = rand(1, 90, 64).requires_grad_(), rand(2, 48, 64).requires_grad_(), rand(3, 48, 64).requires_grad_()
    bg, bu = rand(4, 48).requires_grad_(), rand(5, 48).requires_grad_()
    for half in (F16, BF):
        with torch.autocast("cuda", dtype=half):
            h = gated_linear(x, wg, wu, bg, bu)
        assert h.dtype == half
        dh = rand(6, 90, 48, dtype=half)
        grads = torch.autograd.grad(h, [x, wg, wu, bg, bu], dh)
        assert all(g.dtype == F32 for g in grads)
        r = [t.detach().to(half) for t in (x, wg, wu)]
        det = (*r, bg.detach(), bu.detach())
        check_h(h, *gated_ref(*det, "silu"), "silu", half)
        rounded = list(grads)
        rounded[0] = rounded[0].to(half)  # dx is computed in 16 bits and returned in x's type
        assert torch.equal(rounded[0].float(), grads[0])
        check_grads(*det, "silu", dh, rounded, half, wdtype=F32)


def test_backward_on_either_thread():
    x, wg, wu, w = rand(1, 300, 128, dtype=BF), rand(2, 96, 128, dtype=BF), rand(3, 96, 128, dtype=BF), rand(4, 128)
    dh = rand(5, 300, 96, dtype=BF)
    got = []
    for threads in (False, True):
        with torch.autograd.set_multithreading_enabled(threads):
            leaves = [t.clone().requires_grad_() for t in (x, w, wg, wu)]
            got.append(torch.autograd.grad(gated_linear(rms_norm(*leaves[:2]), *leaves[2:]), leaves, dh))
    assert not torch._C._is_multithreading_enabled()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_deterministic():
    x, wg, wu, dh = rand(1, 3000, 128, dtype=BF), rand(2, 96, 128, dtype=BF), rand(3, 96, 128, dtype=BF), rand(4, 3000, 96, dtype=BF)
    b = rand(5, 96)
    first = _hip.gated_linear_bwd(x, wg, wu, dh, b, b)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, _hip.gated_linear_bwd(x, wg, wu, dh, b, b)))
    w = rand(6, 128)
    _, _, rho = _hip.rms_norm(x, w, stats=True)
    one = _hip.rms_norm_bwd(x, w, rho, x)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(one, _hip.rms_norm_bwd(x, w, rho, x)))


# ------------------------------------------------------------------------------------------ clip
def clip_ref(grads, max_norm, p, inv):
    total = [g.double().abs() for g in grads if g.numel()]
    if p == math.inf:
        n = max(float(t.max()) for t in total)
    else:
        n = math.fsum(float(t.pow(p).sum()) for t in total) ** (1 / p)
    n *= abs(inv)
    return n, min(1.0, max_norm / (n + 1e-6)) * inv


def check_clip(grads, before, norm, outs, max_norm, p, inv=1.0):
    n, c = clip_ref(before, max_norm, p, inv)
    assert abs(float(norm) - n) <= 2 * R * n  # fp64, rounded once
    for g, o in zip(before, outs):
        want = g.double() * c
        within(o, want, 2.1 * R * want.abs() + U[o.dtype] * want.abs() + TINY[o.dtype], "clipped")


@pytest.mark.parametrize("p", [1, 2, math.inf])
@pytest.mark.parametrize("types", [[F32], [BF], [F16], [F32, BF, F16]])
def test_clip(p, types):
    sizes = [1, 7, 2048, 2049, 5000, 3, 0, 70001, 128, 640]
    for max_norm in (0.25, 1e6):
        grads = [rand(i, n, dtype=types[i % len(types)], scale=10.0 ** (i % 4 - 3)) for i, n in enumerate(sizes)]
        before = [g.clone() for g in grads]
        norm = clip_grads(grads, max_norm, p)
        check_clip(grads, before, norm, grads, max_norm, p)
        if max_norm > 1:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))
        outs = [torch.full(g.shape, math.nan, device="cuda", dtype=F32 if i % 2 else g.dtype) for i, g in enumerate(before)]
        inv = torch.full((1,), 1 / 512, device="cuda")
        norm = clip_grads(before, max_norm, p, inv_scale=inv, out=outs)
        check_clip(grads, before, norm, outs, max_norm, p, 1 / 512)


@pytest.mark.parametrize("count,n", [(1, 1), (127, 50), (128, 50), (129, 50), (400, 3000), (3, 3_000_001)])
def test_clip_counts(count, n):
    flat = rand(1, count * n + 1)[1:]  # views of one buffer, off 16-byte boundaries
    grads = [flat[i * n:(i + 1) * n] for i in range(count)]
    before = [g.clone() for g in grads]
    norm = clip_grads(grads, 1.0)
    check_clip(grads, before, norm, grads, 1.0, 2)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_clip_range(dtype):
    """Values whose squares underflow or overflow fp32 (bf16), in the same groups as others; fp16's whole range."""
    tiny, huge = (2.0 ** -120, 2.0 ** 100) if dtype == BF else (2.0 ** -24, 2.0 ** 15)
    for top in (1.0, tiny, huge):
        g = rand(1, 50_000, dtype=F32).abs().clamp(0.5, 1.5)
        g = torch.where(torch.arange(50_000, device="cuda") % 7 == 3, g * top, g * tiny).to(dtype)
        n = float(g.double().square().sum().sqrt())
        assert abs(float(clip_grads([g.clone()], math.inf)) - n) <= 2 * R * n
    g = torch.zeros(50_000, device="cuda", dtype=dtype)
    g[9] = tiny
    assert float(clip_grads([g], math.inf)) == tiny


def test_clip_as_torch_does():
    params = [torch.nn.Parameter(rand(i, *s)) for i, s in enumerate([(64, 32), (64,), (3, 5, 7), (1,)])]
    for scale in (1e-4, 1.0):
        ours, theirs = [], []
        for i, q in enumerate(params):
            q.grad = rand(10 + i, *q.shape, scale=scale)
            theirs.append(torch.nn.Parameter(q.detach().clone()))
            theirs[-1].grad = q.grad.clone()
        params[2].grad = params[2].grad.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # dense, another order
        v = params[0].grad._version
        a = clip_grad_norm_(params + [torch.nn.Parameter(rand(0, 2))], 1.0)
        b = torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        assert params[0].grad._version > v
        torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
        for q, t in zip(params, theirs):
            torch.testing.assert_close(q.grad, t.grad, rtol=4e-7, atol=0)  # both norms within a few 2^-24


def test_clip_not_finite():
    for bad, p in ((math.nan, 2), (math.inf, 2), (math.nan, math.inf), (math.inf, 1)):
        grads = [rand(1, 100), rand(2, 3000, dtype=F16)]
        grads[1][7] = bad
        before = [g.clone() for g in grads]
        with pytest.raises(RuntimeError, match="not clipped"):
            clip_grads(grads, 1.0, p, error_if_nonfinite=True)
        assert torch.equal(grads[0], before[0])
        norm = float(clip_grads(grads, 1.0, p))
        if math.isnan(bad):
            assert math.isnan(norm) and bool(torch.isnan(grads[0]).all())
        else:
            assert math.isinf(norm) and not bool(grads[0].any()) and math.isnan(float(grads[1][7]))
    zero = [torch.zeros(10, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(clip_grads(zero, 1.0)) == 0 and not bool(zero[0].any())
    assert float(clip_grads([zero[1]], 1.0)) == 0
    big = [torch.full((4,), 3e38, device="cuda")]  # squares past fp32
    assert math.isclose(float(clip_grads(big, 1.0, math.inf)), 3e38, rel_tol=1e-6)
    big = [torch.full((4,), 1e30, device="cuda")]
    assert math.isclose(float(clip_grads(big, 1.0)), 2e30, rel_tol=1e-6)
    assert math.isclose(float(big[0].norm()), 1.0, rel_tol=1e-5)


# ------------------------------------------------------------------------------------------ together
class Block(torch.nn.Module):
    def __init__(self, dim, hidden):
        super().__init__()
        self.norm, self.ff, self.down = RMSNorm(dim), GatedLinear(dim, hidden), torch.nn.Linear(hidden, dim)

    def forward(self, x, delta):
        n, s = self.norm(x, delta)
        return s, torch.nn.functional.linear(self.ff(n), self.down.weight, self.down.bias)


def run_blocks(blocks, x, target):
    s, d = x, torch.zeros_like(x)
    for b in blocks:
        s, d = b(s, d)
    loss = ((s + d) - target).square().mean()
    grads = torch.autograd.grad(loss, [p for b in blocks for p in b.parameters()])
    return loss, grads


class PlainBlock(Block):
    def forward(self, x, delta):
        s = x + delta
        n = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * self.norm.weight
        h = torch.nn.functional.silu(self.ff.gate(n)) * self.ff.up(n)
        return s, self.down(h)


def test_blocks_together():
    """Two blocks and the clipping of their gradients, against the same network in 64 bits.  fp32: each value
    passes at most a few thousand roundings of 2^-24, so 1e-4 of a gradient's norm is ample and 1e-2 of a
    wrong term is not."""
    torch.manual_seed(0)
    blocks = [Block(96, 160).cuda() for _ in range(2)]
    plain = [PlainBlock(96, 160) for _ in range(2)]
    for a, b in zip(blocks, plain):
        b.load_state_dict(a.state_dict())
        b.double().cuda()
    x, target = rand(1, 500, 96), rand(2, 500, 96, scale=50)
    loss, grads = run_blocks(blocks, x, target)
    want_loss, want = run_blocks(plain, x.double(), target.double())
    loss, want_loss = loss.detach(), want_loss.detach()
    assert abs(float(loss) - float(want_loss)) < 1e-5 * float(want_loss)
    for g, w in zip(grads, want):
        assert float((g.double() - w).norm()) < 1e-4 * float(w.norm())
    grads = [g.contiguous() for g in grads]
    before = [g.clone() for g in grads]
    norm = clip_grads(grads, 1.0)
    assert float(norm) > 1
    check_clip(grads, before, norm, grads, 1.0, 2)
    with torch.no_grad():  # serving in 8 bits: the norm's output is what the product reads
        b = blocks[0]
        q, sc, s = rms_norm_quant(x.to(BF), b.norm.weight, target.to(BF))
        wg, wu = quant_rows(b.ff.gate.weight), quant_rows(b.ff.up.weight)
        h8 = gated_linear_quant(q, sc, *wg, *wu, b.ff.gate.bias, b.ff.up.bias)
        h = gated_linear(rms_norm(s, b.norm.weight), b.ff.gate.weight.to(BF), b.ff.up.weight.to(BF), b.ff.gate.bias, b.ff.up.bias)
        # e4m3 operands: 2^-4 / sqrt(3) of a value each, three roundings of them in a product pair
        assert float((h8.float() - h.float()).norm()) < 0.08 * float(h.float().norm())


def test_other_streams():
    x, wg, wu, w = rand(1, 2000, 256, dtype=BF), rand(2, 512, 256, dtype=BF), rand(3, 512, 256, dtype=BF), rand(4, 256, dtype=BF)
    r = rand(5, 2000, 256, dtype=BF)

    def work():
        n, s = rms_norm(x, w, r)
        h = gated_linear(n, wg, wu)
        g = [h[:1000].clone(), h[1000:].clone()]
        return [s, h, clip_grads(g, 1.0), *g]

    want = work()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_two_threads():
    """The same calls from two threads at a time, each on a stream of its own, gradients included."""
    import threading

    x, wg, wu, w = rand(1, 3000, 256, dtype=BF), rand(2, 512, 256, dtype=BF), rand(3, 512, 256, dtype=BF), rand(4, 256, dtype=BF)
    dh = rand(5, 3000, 512, dtype=BF)

    def work():
        leaves = [t.detach().requires_grad_() for t in (x, w, wg, wu)]
        grads = torch.autograd.grad(gated_linear(rms_norm(*leaves[:2]), *leaves[2:]), leaves, dh)
        grads = [g.clone() for g in grads]
        return [clip_grads(grads, 1.0), *grads]

    want, got = work(), {}
    torch.cuda.synchronize()

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[k] = [work() for _ in range(4)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_graph():
    """Forward, gradients and clipping captured together, replayed on new inputs, two graphs in turn."""
    D, F, M = 200, 136, 700  # rows of whole 16-byte pieces, ragged tiles

    def make(seed):
        t = dict(x=rand(seed, M, D, dtype=F16), r=rand(seed + 1, M, D, dtype=F16), w=rand(seed + 2, D) + 1,
                 wg=rand(seed + 3, F, D, dtype=F16, scale=0.1), wu=rand(seed + 4, F, D, dtype=F16, scale=0.1),
                 b=rand(seed + 5, F), dh=rand(seed + 6, M, F, dtype=F16), inv=torch.full((1,), 0.5, device="cuda"))
        return t

    def work(t):
        n, s, rho = _hip.rms_norm(t["x"], t["w"], t["r"], stats=True)
        h = _hip.gated_linear(n, t["wg"], t["wu"], t["b"], t["b"], "gelu")
        g = list(_hip.gated_linear_bwd(n, t["wg"], t["wu"], t["dh"], t["b"], t["b"], "gelu"))
        g += list(_hip.rms_norm_bwd(s, t["w"], rho, g.pop(0), s))
        q = _hip.rms_norm_quant(t["x"], t["w"])
        clipped = [torch.empty_like(v) for v in g]
        return [h, *g, _hip.grad_clip(g, 1.0, 2.0, t["inv"], clipped), *clipped, q[0].float(), q[1]]

    states = [make(1), make(100)]
    graphs = []
    for t in states:
        work(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(t)
        graphs.append((graph, out))
    for k in range(4):
        for t in states:
            for name, v in make(1000 * k + int(t["inv"].numel()) + 17 * k).items():
                if name != "inv":
                    t[name].copy_(v)
        for (graph, out), t in zip(graphs, states):
            graph.replay()
        torch.cuda.synchronize()
        for (graph, out), t in zip(graphs, states):
            for a, b in zip(out, work(t)):
                assert torch.equal(a, b)


def test_graph_with_autograd():
    """A block's forward and backward through autograd, captured, replayed between eager passes of the same leaves."""
    torch.manual_seed(0)
    block = Block(256, 512).cuda()
    params = list(block.parameters())
    x, d, dy = (rand(i, 2500, 256, dtype=F32) for i in (1, 2, 3))

    def work():
        with torch.autocast("cuda", dtype=F16):
            s, o = block(x, d)
        return [s.detach(), o.detach(), *torch.autograd.grad([s, o], params, [dy, dy.to(o.dtype)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        for i, t in enumerate((x, d, dy)):
            t.copy_(rand(10 * k + i, 2500, 256))
        with torch.no_grad():
            block.ff.gate.weight.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, work()):
            assert torch.equal(a, b)


def test_modules_train():
    """Gradients through the modules, in place into .grad, next to torch's own layers; no second derivatives."""
    block = Block(64, 96).cuda()
    x = rand(1, 30, 64).requires_grad_()
    s, d = block(x, torch.zeros_like(x))
    (s + d).square().sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in block.parameters())
    y = rms_norm(x, block.norm.weight)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    assert set(block.state_dict()) == {"norm.weight", "ff.gate.weight", "ff.gate.bias", "ff.up.weight", "ff.up.bias",
                                       "down.weight", "down.bias"}
