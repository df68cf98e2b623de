"""GPU checks of the head layers (model/layers.py, csrc/linear.hip,
csrc/norm.hip) against plain implementations in float64.

Tolerances are bounds, not fits.  With u the half step of the output's type
(2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and v = 2^-24 of the float32 sums:
* a sum of n products in any order is within (n + 4) v sum |a b|;
* the output's rounding adds u |y| (and half the spacing of fp16's
  subnormals, 2^-25);
* an activation stretches what enters it by at most 1.13 (the largest slope
  of the five) and is itself evaluated in float32 to 32 v (1 + |z|), its slope
  to 32 v (1 + |z|);
* the gradient of the pre-activation is rounded to the type before it enters
  the products, which adds u |dz| to each factor.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [F32, F16, BF16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
V = 2.0 ** -24


def unit(dt):
    return torch.finfo(dt).eps / 2


def sub(dt):
    return 2.0 ** -25 if dt == F16 else 0.0


@pytest.fixture(scope="module")
def L(mdx):
    from moseq2_detectron_extract_amd.model import layers
    with torch.no_grad():
        yield layers


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def strided(t, pad=0, lead=0):
    """t on the GPU as the middle columns of a wider buffer of NaN, starting
    `lead` elements into it: what lies beside the rows must not be used."""
    buf = torch.full((t.shape[0], lead + t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
    buf[:, lead:lead + t.shape[1]] = t.cuda()
    return buf[:, lead:lead + t.shape[1]]


def within(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), tuple(bad.nonzero()[0].tolist()), (got - want).abs().max().item(),
                           float((tol + 0 * want).max()))


def value(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, act):
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        y = value(z, act)
        (d,) = torch.autograd.grad(y.sum(), z)
    return torch.where(z > 0, 1.0, 0.0).double() if act == "relu" else d


def check_forward(y, pre, x, w, b, r, act, dt):
    x, w = x.double().cpu(), w.double().cpu()
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    for t in (b, r):
        if t is not None:
            z, s = z + t.double().cpu(), s + t.double().cpu().abs()
    ez = (x.shape[1] + 4) * V * s
    if pre is not None:
        within(pre, z, ez + unit(dt) * (z.abs() + ez) + sub(dt), "pre")
    want = value(z, act)
    e = 1.13 * ez + (32 * V * (1 + z.abs()) if act not in ("none", "relu") else 0)
    within(y, want, e + unit(dt) * (want.abs() + e) + sub(dt), "y")


def check_backward(got, dy, x, w, z, act, dt, bias=True, residual=True):
    dy, x, w = dy.double().cpu(), x.double().cpu(), w.double().cpu()
    dz, ez, u = dy, torch.zeros_like(dy), 0.0
    if act != "none":
        z = z.double().cpu()
        dz, u = dy * slope(z, act), unit(dt)
        ez = 32 * V * (1 + z.abs()) * dy.abs() if act != "relu" else ez
    er = ez + u * (dz.abs() + ez) + (sub(dt) if u else 0)  # of dz as it enters the products
    dx = dz @ w
    e = er @ w.abs() + (w.shape[0] + 4) * V * ((dz.abs() + er) @ w.abs())
    within(got.x, dx, e + unit(dt) * (dx.abs() + e) + sub(dt), "dx")
    dw = dz.t() @ x
    e = er.t() @ x.abs() + (x.shape[0] + 4) * V * ((dz.abs() + er).t() @ x.abs())
    within(got.weight, dw, e + unit(dt) * (dw.abs() + e) + sub(dt), "dw")
    if bias:
        within(got.bias, dz.sum(0), ez.sum(0) + (x.shape[0] + 4) * V * (dz.abs() + ez).sum(0), "db")
    if residual:
        within(got.residual, dz, er, "dr")


# M, N, K, pad, lead: one element to several tiles, each edge of the 128-wide
# tiles and the 16-byte pieces, rows at any alignment
SHAPES = [
    (1, 1, 1, 0, 0), (1, 6, 1024, 0, 0), (4, 1024, 256, 0, 0), (3, 17, 5, 1, 0), (16, 16, 64, 0, 0), (17, 33, 65, 3, 1),
    (64, 128, 128, 0, 0), (65, 130, 96, 8, 8), (128, 127, 63, 0, 0), (130, 129, 257, 5, 2), (256, 256, 512, 0, 0),
    (300, 260, 72, 8, 0), (257, 72, 520, 8, 8), (515, 384, 192, 0, 0), (1, 1000, 3001, 7, 0), (33, 64, 4096, 0, 0),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear(L, dt, shape):
    M, N, K, pad, lead = shape
    g = gen(M + 7 * N + 31 * K)
    x, w = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5)
    b, r = normal(g, N), normal(g, M, N, dtype=dt)
    xd, wd, rd = strided(x, pad, lead), strided(w, pad, lead), strided(r, pad, lead)
    act = ACTS[(M + N + K) % 5]
    y, pre = L.linear(xd, wd, b.cuda(), rd, act, return_pre=True)
    check_forward(y, pre, x, w, b, r, act, dt)
    y2 = L.linear(xd, wd)
    check_forward(y2, None, x, w, None, None, "none", dt)
    # into rows of a wider buffer, whose other columns stay as they are
    out = strided(torch.zeros(M, N, dtype=dt), 5, 3)
    base = out._base
    y3 = L.linear(xd, wd, b.cuda(), rd, act, out=out)
    assert y3 is out and torch.equal(out, y)
    assert base[:, :3].isnan().all() and base[:, 3 + N:].isnan().all()
    # over its own residual
    rr = rd.clone()
    assert torch.equal(L.linear(xd, wd, b.cuda(), rr, act, out=rr), y)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(L, dt, act):
    """Every activation over its whole range, its pole-free far ends too."""
    z = torch.cat([torch.linspace(-12, 12, 2049), torch.tensor([-300., -60, -30, 0, -0.0, 30, 60, 300])]).to(dt)
    x, w = z[:, None].contiguous(), torch.ones(1, 1, dtype=dt)
    y, pre = L.linear(x.cuda(), w.cuda(), None, None, act, return_pre=True)
    assert torch.equal(pre.cpu(), x)
    check_forward(y, None, x, w, None, None, act, dt)
    dy = normal(gen(5), len(z), 1, dtype=dt)
    got = L.linear_backward(dy.cuda(), x.cuda(), w.cuda(), pre, act, need_bias=True, need_residual=True)
    check_backward(got, dy, x, w, z[:, None], act, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_backward(L, dt, shape):
    M, N, K, pad, lead = shape
    g = gen(M + 7 * N + 31 * K + 1)
    x, w = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5)
    dy, z = normal(g, M, N, dtype=dt), normal(g, M, N, dtype=dt)
    act = ACTS[(M + N + K + 2) % 5]
    a = [strided(t, pad, lead) for t in (dy, x, w, z)]
    got = L.linear_backward(*a, act, need_bias=True, need_residual=True)
    check_backward(got, dy, x, w, z, act, dt)
    none = L.linear_backward(a[0], a[1], a[2], need_bias=True)
    check_backward(none, dy, x, w, None, "none", dt, residual=False)
    # each gradient alone is the same one
    for k, name in enumerate(("x", "weight", "bias", "residual")):
        need = {f"need_{n}": n == name for n in ("x", "weight", "bias", "residual")}
        one = L.linear_backward(*a, act, **need)
        assert torch.equal(one[k], got[k]) and all(o is None for i, o in enumerate(one) if i != k)


# T, E, N, K, counts: idle groups at either end and in the middle, one group
# with all rows, rows behind the last group, single rows
GROUPS = [
    (1, 1, 5, 9, [1]), (7, 3, 16, 64, [0, 7, 0]), (200, 4, 130, 96, [129, 0, 3, 60]), (64, 8, 256, 128, [8] * 8),
    (300, 5, 64, 65, [1, 128, 127, 0, 2]), (40, 70, 33, 40, [1] * 30 + [0] * 39 + [4]), (513, 2, 257, 72, [256, 257]),
    (9, 4, 24, 16, [0, 0, 0, 0]), (700, 6, 72, 264, [100, 5, 300, 0, 17, 33]), (1030, 3, 256, 512, [513, 260, 257]),
]


def spans(counts, T):
    out, at = [], 0
    for c in counts:
        n = max(0, min(c, T - at))
        out.append((at, at + n))
        at += n
    return out, at


def grouped_inputs(T, E, N, K, dt, seed):
    g = gen(seed)
    return (normal(g, T, K, dtype=dt), normal(g, E, N, K, dtype=dt, scale=K ** -0.5), normal(g, E, N),
            normal(g, T, N, dtype=dt), normal(g, T, N, dtype=dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", GROUPS)
def test_grouped_linear(L, dt, case):
    T, E, N, K, counts = case
    x, w, b, r, _ = grouped_inputs(T, E, N, K, dt, T + E + N)
    sp, end = spans(counts, T)
    x[end:] = float("nan")  # rows of no group are never used
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    act = ACTS[(T + E) % 5]
    args = (strided(x, 3, 1), cd, w.cuda(), b.cuda(), strided(r, 2, 0), act)
    y, pre = L.grouped_linear(*args, return_pre=True)
    for e, (s, t) in enumerate(sp):
        check_forward(y[s:t], pre[s:t], x[s:t], w[e], b[e], r[s:t], act, dt)
    assert (y[end:] == 0).all() and (pre[end:] == 0).all()
    out = torch.full((T, N), 7.0, dtype=dt, device="cuda")
    y2, pre2 = L.grouped_linear(*args, return_pre=True, out=out)
    assert y2 is out and torch.equal(out[:end], y[:end]) and (out[end:] == 7).all() and torch.equal(pre, pre2)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", GROUPS)
def test_grouped_linear_backward(L, dt, case):
    T, E, N, K, counts = case
    x, w, _, z, dy = grouped_inputs(T, E, N, K, dt, T + E + N + 1)
    sp, end = spans(counts, T)
    for t in (x, z, dy):
        t[end:] = float("nan")
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for act in ("none", ACTS[1 + (T + E) % 4]):
        got = L.grouped_linear_backward(strided(dy, 1, 2), strided(x, 3, 1), cd, w.cuda(), strided(z, 8, 0), act,
                                        need_bias=True, need_residual=True)
        for e, (s, t) in enumerate(sp):
            one = L_grads(got, e, s, t)
            check_backward(one, dy[s:t], x[s:t], w[e], z[s:t], act, dt)
            if s == t:
                assert (one.weight == 0).all() and (one.bias == 0).all()
        assert (got.x[end:] == 0).all() and (got.residual[end:] == 0).all()


def L_grads(got, e, s, t):
    return type(got)(got.x[s:t], got.weight[e], got.bias[e], got.residual[s:t])


@pytest.mark.parametrize("counts,same", [([5, -3, 4], [5, 0, 4]), ([4, 9, 9], [4, 8, 0]), ([100, 1, 1], [12, 0, 0]),
                                         ([2 ** 31 - 1, 2 ** 31 - 1, 5], [12, 0, 0]), ([-2 ** 31, 3, 0], [0, 3, 0])])
def test_grouped_linear_bad_counts(L, counts, same):
    """Counts that do not fit the rows are cut to those that do."""
    T, E, N, K = 12, 3, 20, 24
    x, w, b, z, dy = grouped_inputs(T, E, N, K, BF16, 3)
    x, w, b, z, dy = (t.cuda() for t in (x, w, b, z, dy))
    c1, c2 = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in (counts, same))
    assert torch.equal(L.grouped_linear(x, c1, w, b), L.grouped_linear(x, c2, w, b))
    g1, g2 = (L.grouped_linear_backward(dy, x, c, w, z, "silu", need_bias=True, need_residual=True) for c in (c1, c2))
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))


def test_one_group_is_linear(L):
    """The grouped layer with one full group is the linear layer."""
    g = gen(8)
    x, w, b = normal(g, 300, 200, dtype=BF16).cuda(), normal(g, 1, 140, 200, dtype=BF16).cuda(), normal(g, 1, 140).cuda()
    c = torch.tensor([300], dtype=torch.int32, device="cuda")
    y = L.grouped_linear(x, c, w, b, activation="gelu")
    want = L.linear(x, w[0], b[0], activation="gelu")
    within(y, want.cpu(), 2 * unit(BF16) * want.abs().double().cpu() + 1e-5)


def test_empty_rows(L):
    x, w, b = torch.zeros(0, 8, dtype=BF16, device="cuda"), torch.ones(3, 8, dtype=BF16, device="cuda"), torch.ones(3, device="cuda")
    assert L.linear(x, w, b).shape == (0, 3)
    got = L.linear_backward(torch.zeros(0, 3, dtype=BF16, device="cuda"), x, w, need_bias=True)
    assert got.x.shape == (0, 8) and (got.weight == 0).all() and (got.bias == 0).all()
    c = torch.zeros(2, dtype=torch.int32, device="cuda")
    w2 = w.expand(2, 3, 8).contiguous()
    assert L.grouped_linear(x, c, w2).shape == (0, 3)
    got = L.grouped_linear_backward(torch.zeros(0, 3, dtype=BF16, device="cuda"), x, c, w2, need_bias=True)
    assert got.x.shape == (0, 8) and (got.weight == 0).all() and (got.bias == 0).all()
    y, m, r = L.layer_norm(x, return_stats=True)
    assert y.shape == (0, 8) and m.shape == (0,)
    n = L.layer_norm_backward(x, x, m, r)
    assert n.x.shape == (0, 8) and (n.weight == 0).all() and (n.bias == 0).all()


def test_leading_axes_and_layouts(L):
    g = gen(9)
    x = normal(g, 3, 5, 7, 24, dtype=F16).cuda()
    w = normal(g, 10, 24, dtype=F16).cuda()
    want = L.linear(x.view(-1, 24), w).view(3, 5, 7, 10)
    assert torch.equal(L.linear(x, w), want)
    assert torch.equal(L.linear(x, w.t().contiguous().t()), want)              # a transposed weight
    t = x.transpose(0, 2).contiguous().transpose(0, 2)                         # no row view: copied
    assert torch.equal(L.linear(t, w), want)
    assert torch.equal(L.linear(x[0, 0, 0], w), want[0, 0, 0])                 # a single vector
    e = x[:1, :1, :1].expand(2, 3, 4, 24)                                      # rows at distance 0
    assert torch.equal(L.linear(e, w), want[:1, :1, :1].expand(2, 3, 4, 10))
    assert torch.equal(L.layer_norm(t), L.layer_norm(x))


def test_shared_memory_is_refused(L):
    buf = torch.zeros(8, 40, dtype=BF16, device="cuda")
    w = torch.zeros(16, 16, dtype=BF16, device="cuda")
    x = buf[:, :16]
    with pytest.raises(ValueError, match="shares"):
        L.linear(x, w, out=x)
    with pytest.raises(ValueError, match="shares"):
        L.linear(x, w, out=buf[:, 8:24])
    with pytest.raises(ValueError, match="shares"):
        L.linear(torch.ones(8, 16, dtype=BF16, device="cuda"), w, None, buf[:, :16], out=buf[:, 1:17])
    with pytest.raises(ValueError, match="rows"):
        L.linear(x, w, out=torch.zeros(16, 8, dtype=BF16, device="cuda").t())
    with pytest.raises(ValueError, match="shares"):
        L.layer_norm(buf[:, :16], out=buf[:, 1:17])
    L.linear(x, w, out=buf[:, 16:32])  # beside each other


def test_nan_stays_in_its_row(L):
    """A NaN or infinity of one row reaches that row's outputs only, and a
    closed ReLU drops an infinite gradient."""
    g = gen(10)
    x, w = normal(g, 200, 72, dtype=BF16), normal(g, 40, 72, dtype=BF16)
    x[17, 3], x[190, 71] = float("nan"), float("inf")
    y = L.linear(x.cuda(), w.cuda(), activation="relu")
    assert y[17].isnan().all()
    keep = [i for i in range(200) if i not in (17, 190)]
    clean = x.clone()
    clean[[17, 190]] = 0
    assert torch.equal(y[keep], L.linear(clean.cuda(), w.cuda(), activation="relu")[keep])
    z, dy = torch.full((4, 40), -1.0, dtype=BF16).cuda(), torch.full((4, 40), float("inf"), dtype=BF16).cuda()
    got = L.linear_backward(dy, x[:4].cuda(), w.cuda(), z, "relu", need_bias=True, need_residual=True)
    assert all((t == 0).all() for t in got)
    n = L.layer_norm(x.cuda())
    assert n[17].isnan().all() and not n[keep].isnan().any()


NORMS = [(1, 1, 0, 0), (3, 7, 1, 0), (5, 8, 0, 0), (37, 64, 0, 0), (19, 128, 8, 8), (70, 129, 3, 1), (33, 256, 0, 0),
         (9, 257, 7, 2), (21, 512, 0, 0), (40, 1000, 0, 0), (13, 1024, 8, 0), (11, 1025, 1, 1), (6, 2048, 0, 0),
         (5, 4096, 0, 0), (3, 4097, 3, 0), (4, 8192, 0, 0), (3, 12544, 0, 0), (2, 16383, 1, 1), (2, 16384, 0, 0),
         (18, 20001, 1, 0), (2, 65536, 0, 0)]


def norm_inputs(R, D, dt, seed):
    g = gen(seed)
    x = normal(g, R, D, dtype=F32, scale=1.5) + 0.7
    if R > 2:
        x[1] = 3.25           # variance zero
        x[2] = x[2] * 1e-3    # variance near eps
    return x.to(dt), normal(g, D) + 1, normal(g, D), normal(g, R, D, dtype=dt)


def chain(D):
    """Longest chain of additions of a row's sum: a thread's own elements, the
    lanes, the waves."""
    return 64 + D // 1024


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", NORMS)
def test_layer_norm(L, dt, shape):
    R, D, pad, lead = shape
    x, w, b, _ = norm_inputs(R, D, dt, R + D)
    eps = 1e-5
    xd = strided(x, pad, lead)
    y, mean, rstd = L.layer_norm(xd, w.cuda(), b.cuda(), eps, return_stats=True)
    X, c = x.double(), chain(D) * V
    m = X.mean(1)
    d = X - m[:, None]
    rs = (d.square().mean(1) + eps).rsqrt()
    em = c * X.abs().mean(1)
    within(mean, m, em + V * m.abs(), "mean")
    # the computed mean is off by em: the sum of squares grows by D em^2, each
    # deviation is rounded, and the sum itself is off by c
    ev = (em * rs) ** 2 + 2 * V * (1 + m.abs() * rs) + c + 8 * V
    within(rstd, rs, rs * ev, "rstd")
    h = d * rs[:, None]
    eh = (em * rs)[:, None] + h.abs() * (ev[:, None] + 4 * V)

    def check(got, W, B):
        want = h * W + B
        e = eh * W.abs() + 4 * V * (want.abs() + B.abs())
        within(got, want, e + unit(dt) * (want.abs() + e) + sub(dt), "y")
    check(y, w.double(), b.double())
    check(L.layer_norm(xd, eps=eps), torch.ones(D).double(), torch.zeros(D).double())
    check(L.layer_norm(xd, None, b.cuda(), eps=eps), torch.ones(D).double(), b.double())
    out = strided(torch.zeros(R, D, dtype=dt), 2, 1)
    base = out._base
    assert L.layer_norm(xd, w.cuda(), b.cuda(), eps, out=out) is out and torch.equal(out, y)
    assert base[:, :1].isnan().all() and base[:, 1 + D:].isnan().all()
    xc = xd.clone()
    assert torch.equal(L.layer_norm(xc, w.cuda(), b.cuda(), eps, out=xc), y)  # over its input


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", NORMS)
def test_layer_norm_backward(L, dt, shape):
    R, D, pad, lead = shape
    x, w, _, dy = norm_inputs(R, D, dt, R + D + 1)
    X, DY = x.double(), dy.double()
    mean = X.mean(1).float()
    rstd = (X.var(1, correction=0) + 1e-5).rsqrt().float()
    args = (strided(dy, pad, lead), strided(x, pad, lead), mean.cuda(), rstd.cuda())
    m, rs = mean.double()[:, None], rstd.double()[:, None]
    h = (X - m) * rs
    eh = 2 * V * h.abs()

    def check(got, W):
        d = DY * W
        c = chain(D) * V
        s1, s2 = d.mean(1, keepdim=True), (d * h).mean(1, keepdim=True)
        e1 = (c + 4 * V) * d.abs().mean(1, keepdim=True)
        e2 = (c + 8 * V) * (d * h).abs().mean(1, keepdim=True)
        want = rs * (d - s1 - h * s2)
        e = rs * (e1 + h.abs() * e2 + eh * s2.abs() + 8 * V * (d.abs() + s1.abs() + (h * s2).abs()))
        within(got.x, want, e + unit(dt) * (want.abs() + e) + sub(dt), "dx")
        within(got.weight, (DY * h).sum(0), (R + 8) * V * (DY * h).abs().sum(0), "dgamma")
        within(got.bias, DY.sum(0), (R + 8) * V * DY.abs().sum(0), "dbeta")
    got = L.layer_norm_backward(*args, w.cuda())
    check(got, w.double())
    check(L.layer_norm_backward(*args), torch.ones(D).double())
    for k, name in enumerate(("x", "weight", "bias")):
        one = L.layer_norm_backward(*args, w.cuda(), **{f"need_{n}": n == name for n in ("x", "weight", "bias")})
        assert torch.equal(one[k], got[k]) and all(o is None for i, o in enumerate(one) if i != k)


def test_layer_norm_backward_many_rows(L):
    """More rows than the workgroups take at once."""
    for dt, R, D in ((BF16, 9001, 72), (F32, 5003, 260), (F16, 2100, 1032)):
        x, w, _, dy = norm_inputs(R, D, dt, R)
        y, m, r = L.layer_norm(x.cuda(), w.cuda(), return_stats=True)
        got = L.layer_norm_backward(dy.cuda(), x.cuda(), m, r, w.cuda())
        h = (x.double() - m.double().cpu()[:, None]) * r.double().cpu()[:, None]
        DY = dy.double()
        within(got.weight, (DY * h).sum(0), (R + 8) * V * (DY * h).abs().sum(0), "dgamma")
        within(got.bias, DY.sum(0), (R + 8) * V * DY.abs().sum(0), "dbeta")


def test_gradients_against_differences(L):
    """The gradients (float32) against central differences of the forward
    formulas in float64 along random directions: with step 1e-4 their error is
    below 1e-7 of the terms' size, and the kernels' below 1e-5 of it."""
    g = gen(11)
    M, N, K, h = 13, 11, 19, 1e-4
    x, w, b, r = (normal(g, *s).double() for s in ((M, K), (N, K), (N,), (M, N)))
    dy = normal(g, M, N).double()
    for act in ("gelu", "gelu_tanh", "silu"):
        pre = (x @ w.t() + b + r).float().cuda()
        got = L.linear_backward(dy.float().cuda(), x.float().cuda(), w.float().cuda(), pre, act, need_bias=True,
                                need_residual=True)

        def loss(x, w, b, r):
            return (value(x @ w.t() + b + r, act) * dy).sum()
        for k, t in enumerate((x, w, b, r)):
            v = normal(g, *t.shape).double()
            a = [x, w, b, r]
            hi, lo = list(a), list(a)
            hi[k], lo[k] = t + h * v, t - h * v
            num = (loss(*hi) - loss(*lo)) / (2 * h)
            ana = (got[k].double().cpu() * v).sum()
            size = (got[k].double().cpu() * v).abs().sum()
            assert abs(num - ana) <= 1e-5 * size, (act, k, num, ana)
    gm, bt = normal(g, K).double() + 1, normal(g, K).double()
    gy = normal(g, M, K).double()

    def norm_loss(x, gm, bt):
        d = x - x.mean(1, keepdim=True)
        return ((d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gm + bt) * gy).sum()
    _, m, rs = L.layer_norm(x.float().cuda(), return_stats=True)
    got = L.layer_norm_backward(gy.float().cuda(), x.float().cuda(), m, rs, gm.float().cuda())
    for k, t in enumerate((x, gm, bt)):
        v = normal(g, *t.shape).double()
        hi, lo = [x, gm, bt], [x, gm, bt]
        hi[k], lo[k] = t + h * v, t - h * v
        num = (norm_loss(*hi) - norm_loss(*lo)) / (2 * h)
        ana, size = (got[k].double().cpu() * v).sum(), (got[k].double().cpu() * v).abs().sum()
        assert abs(num - ana) <= 1e-5 * size, (k, num, ana)


def block(L, p, x, counts):
    """norm -> grouped up-projection with GELU -> grouped down-projection on
    the residual -> norm -> predictor, and back."""
    h, m1, r1 = L.layer_norm(x, p["g1"], p["b1"], return_stats=True)
    u, z = L.grouped_linear(h, counts, p["w1"], p["c1"], activation="gelu", return_pre=True)
    o = L.grouped_linear(u, counts, p["w2"], p["c2"], residual=x)
    n, m2, r2 = L.layer_norm(o, p["g2"], p["b2"], return_stats=True)
    y, zy = L.linear(n, p["w3"], p["c3"], activation="silu", return_pre=True)
    return y, (h, m1, r1, u, z, o, n, m2, r2, zy)


def block_backward(L, p, x, counts, saved, dy):
    h, m1, r1, u, z, o, n, m2, r2, zy = saved
    g3 = L.linear_backward(dy, n, p["w3"], zy, "silu", need_bias=True)
    gn2 = L.layer_norm_backward(g3.x, o, m2, r2, p["g2"])
    g2 = L.grouped_linear_backward(gn2.x, u, counts, p["w2"], need_bias=True, need_residual=True)
    g1 = L.grouped_linear_backward(g2.x, h, counts, p["w1"], z, "gelu", need_bias=True)
    gn1 = L.layer_norm_backward(g1.x, x, m1, r1, p["g1"])
    return {"x": gn1.x + g2.residual, "g1": gn1.weight, "b1": gn1.bias, "w1": g1.weight, "c1": g1.bias, "w2": g2.weight,
            "c2": g2.bias, "g2": gn2.weight, "b2": gn2.bias, "w3": g3.weight, "c3": g3.bias}


def block_params(dt, D=40, H=72, P=10, E=3):
    g = gen(12)
    p = {"g1": normal(g, D) * 0.2 + 1, "b1": normal(g, D) * 0.2, "g2": normal(g, D) * 0.2 + 1, "b2": normal(g, D) * 0.2,
         "w1": normal(g, E, H, D, dtype=dt, scale=D ** -0.5), "c1": normal(g, E, H),
         "w2": normal(g, E, D, H, dtype=dt, scale=H ** -0.5), "c2": normal(g, E, D),
         "w3": normal(g, P, D, dtype=dt, scale=D ** -0.5), "c3": normal(g, P)}
    return p, normal(g, 90, D, dtype=dt), normal(g, 90, P, dtype=dt)


def test_block(L):
    """A run of all the layers, forward and backward, in float32 against
    torch's autograd in float64.  Each stage is off by at most some 1e-5 of
    its largest value (bounds above), seven stages by 1e-4."""
    p, x, dy = block_params(F32)
    counts = [40, 0, 50]
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    pd = {k: v.cuda() for k, v in p.items()}
    y, saved = block(L, pd, x.cuda(), cd)
    got = block_backward(L, pd, x.cuda(), cd, saved, dy.cuda())
    with torch.enable_grad():
        q = {k: v.double().requires_grad_() for k, v in p.items()}
        X = x.double().requires_grad_()

        def norm(t, g, b):
            d = t - t.mean(1, keepdim=True)
            return d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * g + b

        def groups(t, w, c):
            return torch.cat([t[s:e] @ w[i].t() + c[i] for i, (s, e) in enumerate(spans(counts, 90)[0])])
        o = X + groups(value(groups(norm(X, q["g1"], q["b1"]), q["w1"], q["c1"]), "gelu"), q["w2"], q["c2"])
        want = value(norm(o, q["g2"], q["b2"]) @ q["w3"].t() + q["c3"], "silu")
        (want * dy.double()).sum().backward()
    within(y, want.detach(), 1e-4 * want.detach().abs().max())
    for k, t in {**q, "x": X}.items():
        within(got[k], t.grad, 1e-4 * t.grad.abs().max(), k)


def test_captured_block(L):
    """The block forward and backward in a graph, replayed on new inputs, with
    eager work between the replays; the counts change too."""
    p, x, dy = block_params(BF16)
    p = {k: v.cuda() for k, v in p.items()}
    xs, dys = x.cuda(), dy.cuda()
    cd = torch.tensor([40, 0, 50], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, s = block(L, p, xs, cd)
        block_backward(L, p, xs, cd, s, dys)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s = block(L, p, xs, cd)
        got = block_backward(L, p, xs, cd, s, dys)
    for k, counts in enumerate(([40, 0, 50], [1, 2, 3], [90, 0, 0], [0, 45, 45])):
        g = gen(20 + k)
        xs.copy_(normal(g, 90, 40, dtype=BF16))
        dys.copy_(normal(g, 90, 10, dtype=BF16))
        cd.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ye, se = block(L, p, xs, cd)
        ge = block_backward(L, p, xs, cd, se, dys)
        assert torch.equal(y, ye) and all(torch.equal(got[n], ge[n]) for n in ge), counts


def test_two_streams_and_repeats(L):
    """Calls on two streams side by side, and repeated calls, give the same
    bits."""
    g = gen(13)
    x, w, dy = normal(g, 700, 2048, dtype=BF16).cuda(), normal(g, 96, 2048, dtype=BF16).cuda(), normal(g, 700, 96, dtype=BF16).cuda()
    z = normal(g, 700, 96, dtype=BF16).cuda()

    def work():
        y = L.linear(x, w, None, None, "gelu")
        got = L.linear_backward(dy, x, w, z, "gelu", need_bias=True)
        n, m, r = L.layer_norm(x, return_stats=True)
        return [y, got.x, got.weight, got.bias, n, *L.layer_norm_backward(x, x, m, r)]
    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(work())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_offsets_past_32_bits(L):
    """Rows whose offset passes 2^31 elements (a wide buffer; only its ends
    are touched)."""
    ld = (1 << 31) // 100
    buf = torch.empty(130 * ld, dtype=F16, device="cuda")
    x = torch.as_strided(buf, (130, 64), (ld, 1))
    g = gen(14)
    v, w = normal(g, 130, 64, dtype=F16), normal(g, 24, 64, dtype=F16, scale=0.1)
    x.copy_(v.cuda())
    assert torch.equal(L.linear(x, w.cuda()), L.linear(v.cuda(), w.cuda()))
    assert torch.equal(L.layer_norm(x), L.layer_norm(v.cuda()))
    c = torch.tensor([100, 30], dtype=torch.int32, device="cuda")
    w2 = torch.stack([w, w * 2]).cuda()
    assert torch.equal(L.grouped_linear(x, c, w2), L.grouped_linear(v.cuda(), c, w2))
    dy = normal(g, 130, 24, dtype=F16).cuda()
    a, b = (L.grouped_linear_backward(dy, t, c, w2, need_bias=True) for t in (x, v.cuda()))
    assert all(torch.equal(p, q) for p, q in zip(a[:3], b[:3]))
    out = torch.as_strided(buf, (130, 24), (ld, 1), storage_offset=128)
    assert torch.equal(L.linear(x, w.cuda(), out=out), L.linear(v.cuda(), w.cuda()))
    assert torch.equal(L.layer_norm(x, out=x), L.layer_norm(v.cuda()))


def test_c_entry_with_less_workspace(L, mdx):
    """mdx_linear without workspace, and with less than it asks for, does not
    split the reduction: the same values to the sums' rounding."""
    from moseq2_detectron_extract_amd._lib import call
    g = gen(15)
    M, N, K = 5, 24, 8192
    x, w = normal(g, M, K, dtype=F32).cuda(), normal(g, N, K, dtype=F32, scale=K ** -0.5).cuda()
    P = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    n = call("mdx_linear_workspace_bytes", M, N, K, 0)
    for nbytes in (0, max(n - 1, 0), n):
        out = torch.empty(M, N, device="cuda")
        ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda")
        call("mdx_linear", P(x), K, P(w), K, None, None, 0, M, N, K, 0, 0, None, 0, P(out), N, P(ws), nbytes, None)
        torch.cuda.synchronize()
        check_forward(out, None, x.cpu(), w.cpu(), None, None, "none", F32)
        if nbytes < n:
            assert (ws == 255).all()


# Shapes of whole and ragged large tiles (256 x 256, 16-bit, aligned rows):
# reductions shorter than the pipeline's four steps of 64, of a whole number of
# steps and not, odd and even numbers of them; grouped ones with short, empty
# and long groups
LARGE = [(4096, 2048, 8), (4104, 2048, 64), (4097, 2056, 136), (2048, 4096, 200), (8200, 1032, 256), (4096, 2048, 328),
         (2300, 4104, 72), (4096, 2048, 648)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", LARGE)
def test_large_tiles(L, dt, shape):
    """Forward and backward where the 256-wide tile has enough work."""
    M, N, K = shape
    g = gen(M + N + K)
    x, w, b = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5), normal(g, N)
    r, dy, z = (normal(g, M, N, dtype=dt) for _ in range(3))
    act = ACTS[1 + (M + K) % 4]
    y, pre = L.linear(x.cuda(), w.cuda(), b.cuda(), r.cuda(), act, return_pre=True)
    check_forward(y, pre, x, w, b, r, act, dt)
    got = L.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda(), act, need_bias=True, need_residual=True)
    check_backward(got, dy, x, w, z, act, dt)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("E,N,K,counts,tail", [
    (6, 2048, 72, [1000, 0, 3, 2000, 256, 700], 100), (3, 4096, 264, [1, 2000, 513], 0),
    (9, 1032, 1024, [300, 0, 0, 900, 1300, 17, 0, 2100, 64], 900), (2, 2048, 128, [0, 4096], 1)])
def test_large_tiles_grouped(L, dt, E, N, K, counts, tail):
    T = sum(counts) + tail
    x, w, b, z, dy = grouped_inputs(T, E, N, K, dt, T + N)
    sp, end = spans(counts, T)
    for t in (x, z, dy):
        t[end:] = float("nan")
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    act = ACTS[1 + T % 4]
    y = L.grouped_linear(x.cuda(), cd, w.cuda(), b.cuda(), None, act)
    got = L.grouped_linear_backward(dy.cuda(), x.cuda(), cd, w.cuda(), z.cuda(), act, need_bias=True, need_residual=True)
    for e, (s, t) in enumerate(sp):
        check_forward(y[s:t], None, x[s:t], w[e], b[e], None, act, dt)
        check_backward(L_grads(got, e, s, t), dy[s:t], x[s:t], w[e], z[s:t], act, dt)
    assert (y[end:] == 0).all() and (got.x[end:] == 0).all() and (got.residual[end:] == 0).all()
    out = torch.full((T, N), 3.0, dtype=dt, device="cuda")
    L.grouped_linear(x.cuda(), cd, w.cuda(), b.cuda(), None, act, out=out)
    assert torch.equal(out[:end], y[:end]) and (out[end:] == 3).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1000, 1024, 1024), (1000, 512, 4096), (2048, 1024, 72), (515, 1040, 2056),
                                   (1001, 515, 1003), (2100, 1031, 263)])
def test_middle_sizes(L, dt, M, N, K):
    """The 64- and 128-wide tiles with whole and split reductions, aligned and not."""
    g = gen(M + N + K)
    x, w, b = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5), normal(g, N)
    dy, z = normal(g, M, N, dtype=dt), normal(g, M, N, dtype=dt)
    act = ACTS[(M + K) % 5]
    y, pre = L.linear(x.cuda(), w.cuda(), b.cuda(), None, act, return_pre=True)
    check_forward(y, pre, x, w, b, None, act, dt)
    got = L.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda(), act, need_bias=True, need_residual=True)
    check_backward(got, dy, x, w, z, act, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [1, 5, 16, 17, 32])
@pytest.mark.parametrize("N,K", [(1024, 12544), (40, 8200), (4100, 264), (2056, 4100), (30, 4099), (33000, 16)])
def test_few_rows(L, dt, M, N, K):
    """Few rows: long reductions in slices, wide weights, odd ends of both."""
    g = gen(M + N + K)
    x, w, b, r = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5), normal(g, N), normal(g, M, N, dtype=dt)
    act = ACTS[(M + K) % 5]
    y, pre = L.linear(strided(x, 3, 1), w.cuda(), b.cuda(), r.cuda(), act, return_pre=True)
    check_forward(y, pre, x, w, b, r, act, dt)


def many_counts(E, g):
    c = torch.randint(0, 4, (E,), generator=g)
    c[torch.randperm(E, generator=g)[:E // 3]] = 0
    c[E // 2] = 300
    return c.tolist()


@pytest.mark.parametrize("E", [63, 64, 65, 200, 1000])
def test_many_groups(L, E):
    """More groups than a wave has lanes, and the edges of that."""
    g = gen(E)
    counts = many_counts(E, g)
    T, N, K, dt = sum(counts) + 3, 24, 40, BF16
    x, w, b, z, dy = grouped_inputs(T, E, N, K, dt, E)
    sp, end = spans(counts, T)
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y = L.grouped_linear(x.cuda(), cd, w.cuda(), b.cuda(), None, "silu")
    got = L.grouped_linear_backward(dy.cuda(), x.cuda(), cd, w.cuda(), z.cuda(), "silu", need_bias=True, need_residual=True)
    y, got = y.cpu(), type(got)(*(t.cpu() for t in got))
    for e, (s, t) in enumerate(sp):
        check_forward(y[s:t], None, x[s:t], w[e], b[e], None, "silu", dt)
        check_backward(L_grads(got, e, s, t), dy[s:t], x[s:t], w[e], z[s:t], "silu", dt)
    assert (y[end:] == 0).all() and (got.x[end:] == 0).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("E,per,N,K", [(4, 1, 40, 1024), (4, 4, 72, 4096), (3, 12, 33, 12544), (3, 13, 40, 12544),
                                       (5, 1, 24, 8191), (8, 16, 264, 520), (8, 17, 264, 520), (70, 1, 48, 2048)])
def test_grouped_few_rows(L, dt, E, per, N, K):
    """Few rows to a group, long reductions and short ones, on both sides of
    where another kernel takes over; one group holds most rows, one none."""
    g = gen(E + per + N + K)
    T = E * per
    counts = [0] * E
    counts[E // 2] = T - T // 4 - 1
    for k in range(T // 4):
        counts[k * 5 % E if k * 5 % E != 1 else 0] += 1
    x, w, b, z, dy = grouped_inputs(T, E, N, K, dt, E + per)
    r = normal(g, T, N, dtype=dt)
    act = ACTS[(E + per) % 5]
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y, pre = L.grouped_linear(strided(x, 8), cd, w.cuda(), b.cuda(), r.cuda(), act, return_pre=True)
    y, pre = y.cpu(), pre.cpu()
    sp, end = spans(counts, T)
    for e, (s, t) in enumerate(sp):
        check_forward(y[s:t], pre[s:t], x[s:t], w[e], b[e], r[s:t], act, dt)
    assert (y[end:] == 0).all() and (pre[end:] == 0).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_far_values(L, dt, act):
    """Arguments near the ends of the type's range: every gate is 0 or 1 there,
    and nothing overflows on the way.  (Rounding: none, 0 and 1 are exact.)"""
    far = [1e4, 6e4] if dt == F16 else [1e4, 1e10, 1e19, 1e20, 3e38]
    z = torch.tensor([-v for v in far] + far, dtype=dt, device="cuda").repeat(3, 5)
    M, N = z.shape
    x, w = torch.zeros(M, 8, dtype=dt, device="cuda"), torch.zeros(N, 8, dtype=dt, device="cuda")
    want = z if act in (None, "none") else z.clamp(min=0)
    assert torch.equal(L.linear(x, w, None, z, act), want)
    got = L.linear_backward(torch.ones_like(z), x, w, z, act, need_residual=True).residual
    assert torch.equal(got, torch.ones_like(z) if act in (None, "none") else (z > 0).to(dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(129, 2048, 0, 0), (1030, 2049, 3, 1), (5, 8193, 0, 0), (300, 12544, 8, 0), (600, 16384, 0, 0),
                                   (2100, 1500, 0, 0), (4100, 130, 1, 1)])
def test_layer_norm_backward_shares(L, dt, shape):
    """Rows on both sides of where more workgroups share the sums."""
    test_layer_norm_backward(L, dt, shape)


def gate(z, act):
    """What z is multiplied with by an activation of z <= 0 or more, to the last digits of the far tails."""
    if act == "gelu":
        return 0.5 * torch.special.erfc(z * -0.5 ** 0.5)
    if act == "gelu_tanh":
        z = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)
    return torch.special.expit(z)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act,low", [("gelu", -12.0), ("gelu_tanh", -9.0), ("silu", -80.0)])
def test_activation_tails(L, dt, act, low):
    """Relative errors: an activation's far negative tail keeps its digits.

    float32: the fits are good to 1e-8, their float32 evaluation to 6 v (emulated), exp2 and the reciprocal
    to one step (2 v) each, of which the latter enters twice, and the product with z adds v: below 16 v.
    16 bits: 2.8e-5 (the fit's 2.2e-5 with its roundings; exponents up to 126 rounded three times to float32
    give 1.6e-5), a few steps of float32 beside it: below 4e-5, and the output's rounding.  The slope is the
    gate and z times the density, each to that."""
    z = torch.cat([torch.linspace(low, 0, 4001), torch.linspace(0, 12, 1001)[1:]]).to(dt)
    Z = z.double()
    t, u = (16 * V, 0.0) if dt == F32 else (4e-5, unit(dt))
    x, w = z[:, None].contiguous().cuda(), torch.ones(1, 1, dtype=dt, device="cuda")
    y = L.linear(x, w, None, None, act)
    want = Z * gate(Z, act)
    within(y[:, 0], want, (t + u) * want.abs() + sub(dt), act)
    s, c = gate(Z, act), gate(-Z, act)
    if act == "gelu":
        part = Z * torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)
    else:
        part = Z * s * c * (1 if act == "silu" else math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * Z * Z))
    got = L.linear_backward(torch.ones_like(x), x, w, x, act, need_x=False, need_weight=False, need_residual=True)
    within(got.residual[:, 0], s + part, t * (s + part.abs()) + u * (s + part).abs() + sub(dt), act)


def test_float16_range_of_dz(L):
    """dz enters the float16 products rounded to float16: past 65504 it is infinite, below 2^-25 zero, and the
    bias's gradient is summed before that.  float32 operands keep both.  Bounds: 4e-5 and 16 v of the slope's
    two parts (test_activation_tails), and v for each product and sum."""
    z = torch.tensor([[1.5, -0.5]], dtype=F16, device="cuda")
    dy = torch.tensor([[65504.0, 2.0 ** -24]], dtype=F16, device="cuda")  # slopes 1.127 and 0.132
    x = torch.full((1, 8), 2.0 ** -10, dtype=F16, device="cuda")
    w = torch.tensor([[2.0 ** -10] * 8, [1.0] * 8], dtype=F16, device="cuda")
    got = L.linear_backward(dy, x, w, z, "gelu", need_bias=True, need_residual=True)
    assert got.residual.tolist() == [[float("inf"), 0.0]] and got.x.isinf().all()
    assert got.weight[0].isinf().all() and (got.weight[1] == 0).all()
    Z, DY, W = z.double().cpu(), dy.double().cpu(), w.double().cpu()
    want, size = DY * slope(Z, "gelu"), DY * (gate(Z, "gelu") + (Z * torch.exp(-Z * Z / 2)).abs() / math.sqrt(2 * math.pi))
    within(got.bias, want[0], (4e-5 + 2 * V) * size[0], "db")
    full = L.linear_backward(dy.float(), x.float(), w.float(), z.float(), "gelu", need_residual=True)
    within(full.residual, want, 18 * V * size, "dr")
    within(full.x, want @ W, 24 * V * (size @ W), "dx")


def test_negative_views(L):
    """Operands that are lazily negated views (a conjugate's imaginary part)."""
    c = torch.view_as_complex(normal(gen(31), 6, 1, 2)).cuda()
    x, plain = c.conj().imag, -c.imag.contiguous()
    assert x.is_neg()
    w, b = torch.full((1, 1), 2.0, device="cuda"), torch.full((1,), 0.5, device="cuda")
    assert torch.equal(L.linear(x, w, b, x), L.linear(plain, w, b, plain))
    n, m = c[:1].conj().imag, -c[:1].imag.contiguous()  # (1, 1): also contiguous
    assert n.is_neg() and n.is_contiguous()
    assert torch.equal(L.linear(n, n, n[0], n), L.linear(m, m, m[0], m))
    for got, want in zip(L.linear_backward(x, x, n, x, "silu", need_bias=True, need_residual=True),
                         L.linear_backward(plain, plain, m, plain, "silu", need_bias=True, need_residual=True)):
        assert torch.equal(got, want)
    assert torch.equal(L.layer_norm(x, n[0], n[0]), L.layer_norm(plain, m[0], m[0]))
    with pytest.raises(ValueError, match="rows"):
        L.linear(plain, w, out=x)


@pytest.mark.parametrize("M", [6 * 10 ** 8, 12 * 10 ** 8])
def test_narrow_outputs_of_many_rows(L, M):
    """The most rows that a launch of the 64-wide tiles has threads for, and more than those: the weight is the
    unit matrix, so that every product is exact."""
    dt = BF16
    x = torch.empty(M, 8, dtype=dt, device="cuda").normal_()
    w = torch.eye(8, dtype=dt, device="cuda")
    assert torch.equal(L.linear(x, w), x)
    assert torch.equal(L.linear_backward(x, x, w, need_weight=False).x, x)


def test_wide_output_of_one_row(L):
    """More columns than the kernel of few rows has threads for."""
    N = 54 * 10 ** 7
    w = torch.empty(N, 8, dtype=BF16, device="cuda").normal_()
    x = torch.zeros(1, 8, dtype=BF16, device="cuda")
    x[0, 3] = 1
    assert torch.equal(L.linear(x, w)[0], w[:, 3])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1000, 512, 4096), (300, 256, 2048), (9, 40, 8192)])
def test_c_entry_splits_whole_or_not(L, mdx, dt, M, N, K):
    """mdx_linear with less workspace than its slices take splits nothing, however little is missing, and leaves
    the workspace as it was; the result does not follow the size."""
    from moseq2_detectron_extract_amd._lib import call
    g = gen(16)
    x, w = normal(g, M, K, dtype=dt).cuda(), normal(g, N, K, dtype=dt, scale=K ** -0.5).cuda()
    P = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    code = {F32: 0, BF16: 3}[dt]
    most = call("mdx_linear_workspace_bytes", M, N, K, code)
    assert most % (4 * M * N) == 0 and most >= 8 * M * N

    def run(nbytes):
        out, ws = torch.empty(M, N, dtype=dt, device="cuda"), torch.full((most,), 255, dtype=torch.uint8, device="cuda")
        call("mdx_linear", P(x), K, P(w), K, None, None, 0, M, N, K, 0, code, None, 0, P(out), N, P(ws), nbytes, None)
        torch.cuda.synchronize()
        check_forward(out, None, x.cpu(), w.cpu(), None, None, "none", dt)
        return out, bool((ws == 255).all())
    whole, untouched = run(most)
    assert not untouched and torch.equal(whole, L.linear(x, w))
    once, untouched = run(0)
    assert untouched
    seen = {}
    for nbytes in range(2 * M * N, most + 1, 2 * M * N):
        for n in (nbytes - 1, nbytes):
            out, untouched = run(n)
            seen[n] = untouched
            assert torch.equal(out, once if untouched else whole), n
    need = min(n for n, u in seen.items() if not u)  # one size on which it turns, that of whole slices
    assert need % (4 * M * N) == 0 and all(u == (n < need) for n, u in seen.items()), seen


# Every kernel of csrc/linear.hip by name (mdx_linear_plan), whole reductions and split ones, each at a shape that
# is given to it: (kernel, split, dtypes, M, N, K).  Odd sizes end inside a tile, a piece and a step.
KERNELS = ["256", "128", "64", "128 any", "64 any", "few"]
HALF = [F16, BF16]


def plan(E, T, N, K, dt, backward):
    from moseq2_detectron_extract_amd._lib import call
    n = 16 // dt.itemsize
    aligned = K % n == 0 and (not backward or N % n == 0)
    p = call("mdx_linear_plan", E, T, N, K, {F32: 0, F16: 1, BF16: 3}[dt], aligned, backward)
    return KERNELS[p % 16], p // 16 > 1


def each_type(cases):
    return [pytest.param(k, split, dt, *shape, id=f"{k}{'-split' if split else ''}-{str(dt)[6:]}-{'x'.join(map(str, shape[:4]))}")
            for k, split, dts, *shape in cases for dt in dts]


@pytest.mark.parametrize("kernel,split,dt,M,N,K", each_type([
    ("256", False, HALF, 2048, 4104, 520), ("256", True, HALF, 1000, 2056, 4104),
    ("128", False, DTYPES, 1000, 2056, 264), ("128", True, [F32], 1000, 1000, 4100),
    ("64", False, DTYPES, 300, 264, 264), ("64", True, DTYPES, 300, 264, 2056),
    ("128 any", False, DTYPES, 4000, 1027, 263), ("128 any", True, HALF, 1001, 1003, 4097),
    ("128 any", True, [F32], 515, 1990, 2047),
    ("64 any", False, DTYPES, 301, 2049, 515), ("64 any", True, DTYPES, 301, 257, 1027),
    ("few", False, DTYPES, 20, 4100, 264), ("few", True, DTYPES, 20, 40, 8200)]))
def test_each_kernel_forward(L, kernel, split, dt, M, N, K):
    assert plan(0, M, N, K, dt, 0) == (kernel, split)
    g = gen(M + N + K)
    x, w, b = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5), normal(g, N)
    r = normal(g, M, N, dtype=dt)
    for act in ("none", ACTS[1 + (M + K) % 4]):
        y, pre = L.linear(x.cuda(), w.cuda(), b.cuda(), r.cuda(), act, return_pre=True)
        check_forward(y, pre, x, w, b, r, act, dt)


@pytest.mark.parametrize("kernel,split,dt,M,N,K", each_type([
    ("256", False, HALF, 2048, 2056, 2088), ("256", True, HALF, 1000, 264, 8200), ("256", True, HALF, 4096, 1024, 1024),
    ("128", False, DTYPES, 300, 264, 4104), ("128", True, [F32], 1000, 264, 4104), ("128", True, HALF, 4000, 1000, 520),
    ("64", False, DTYPES, 300, 264, 520), ("64", True, [F32], 1000, 264, 520), ("64", True, HALF, 2100, 264, 520),
    ("128 any", False, DTYPES, 300, 261, 8195),
    ("128 any", True, DTYPES, 1001, 261, 4097), ("64 any", False, DTYPES, 301, 261, 517),
    ("64 any", True, HALF, 1001, 261, 517), ("64 any", True, [F32], 515, 261, 517)]))
def test_each_kernel_backward(L, kernel, split, dt, M, N, K):
    """Without an activation dz is the gradient itself, so that each product's bound is that of its sum."""
    assert plan(0, M, N, K, dt, 1) == (kernel, split)
    g = gen(M + N + K)
    x, w = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5)
    dy, z = normal(g, M, N, dtype=dt), normal(g, M, N, dtype=dt)
    for act in ("none", ACTS[1 + (M + K) % 4]):
        got = L.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda(), act, need_bias=True, need_residual=True)
        check_backward(got, dy, x, w, z, act, dt)


def uneven(E, T):
    """T rows in E groups: the second empty, the third of one row, the rest growing, the first with most."""
    c = [0, 0, 1] + [k + 1 for k in range(E - 3)] if E > 3 else [0, 0, 1][:E]
    if E > 3:
        c = c[:3] + [v * (T // 3) // sum(c[3:]) for v in c[3:]]
    c[0] = T - sum(c) - 5
    return c


@pytest.mark.parametrize("kernel,split,dt,E,T,N,K", each_type([
    ("256", False, HALF, 3, 4099, 2056, 264), ("128", False, DTYPES, 2, 8195, 264, 264), ("64", False, DTYPES, 4, 1003, 264, 264),
    ("128 any", False, HALF, 3, 4099, 2051, 519),
    ("128 any", False, [F32], 3, 1003, 4001, 263), ("64 any", False, DTYPES, 4, 1003, 261, 263),
    ("few", False, DTYPES, 4, 7, 72, 8200)]))
def test_each_kernel_grouped_forward(L, kernel, split, dt, E, T, N, K):
    assert plan(E, T, N, K, dt, 0) == (kernel, split)
    x, w, b, r, _ = grouped_inputs(T, E, N, K, dt, T + E + N)
    counts = uneven(E, T) if T > 100 else [2, 0, 1, 2]
    sp, end = spans(counts, T)
    x[end:] = float("nan")
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for act in ("none", ACTS[1 + (T + K) % 4]):
        y = L.grouped_linear(x.cuda(), cd, w.cuda(), b.cuda(), r.cuda(), act).cpu()
        for e, (s, t) in enumerate(sp):
            check_forward(y[s:t], None, x[s:t], w[e], b[e], r[s:t], act, dt)
        assert (y[end:] == 0).all()


@pytest.mark.parametrize("kernel,split,dt,E,T,N,K", each_type([
    ("256", False, HALF, 8, 2051, 1032, 1032), ("256", True, HALF, 8, 8192, 264, 520), ("256", True, HALF, 2, 16384, 1024, 512),
    ("128", False, DTYPES, 5, 1003, 264, 1032), ("128", True, [F32], 8, 8192, 256, 512), ("128", True, HALF, 2, 8195, 264, 520),
    ("64", False, DTYPES, 3, 1003, 264, 264), ("64", True, [F32], 2, 2051, 264, 264), ("64", True, HALF, 2, 4099, 264, 264),
    ("128 any", False, HALF, 8, 1003, 515, 521), ("128 any", False, [F32], 5, 1003, 1001, 521),
    ("128 any", True, [F32], 3, 4003, 515, 1031), ("128 any", True, HALF, 2, 4099, 261, 521),
    ("64 any", False, DTYPES, 5, 1003, 261, 263), ("64 any", True, [F32], 2, 2051, 261, 263),
    ("64 any", True, HALF, 2, 2051, 261, 263)]))
def test_each_kernel_grouped_backward(L, kernel, split, dt, E, T, N, K):
    """dW's slices of a group, of an empty one and of one row too, and each gradient alone."""
    assert plan(E, T, N, K, dt, 1) == (kernel, split)
    x, w, _, z, dy = grouped_inputs(T, E, N, K, dt, T + E + N + 1)
    counts = uneven(E, T)
    sp, end = spans(counts, T)
    for t in (x, z, dy):
        t[end:] = float("nan")
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    a = (dy.cuda(), x.cuda(), cd, w.cuda(), z.cuda())
    for act in ("none", ACTS[1 + (T + K) % 4]):
        got = L.grouped_linear_backward(*a, act, need_bias=True, need_residual=True)
        here = type(got)(*(t.cpu() for t in got))
        for e, (s, t) in enumerate(sp):
            check_backward(L_grads(here, e, s, t), dy[s:t], x[s:t], w[e], z[s:t], act, dt)
        assert (here.x[end:] == 0).all() and (here.residual[end:] == 0).all()
        for k, name in enumerate(("x", "weight", "bias", "residual")):
            one = L.grouped_linear_backward(*a, act, **{f"need_{n}": n == name for n in ("x", "weight", "bias", "residual")})
            assert torch.equal(one[k], got[k]) and all(o is None for i, o in enumerate(one) if i != k)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shape", LARGE)
def test_large_shapes_backward(L, dt, shape):
    """The shapes of partial K-tiles backward, with the bound of the products' sums alone."""
    M, N, K = shape
    g = gen(M + N + K + 1)
    x, w, dy = normal(g, M, K, dtype=dt), normal(g, N, K, dtype=dt, scale=K ** -0.5), normal(g, M, N, dtype=dt)
    check_backward(L.linear_backward(dy.cuda(), x.cuda(), w.cuda(), need_bias=True), dy, x, w, None, "none", dt, residual=False)


def test_layer_norm_backward_very_wide(L):
    """More columns than a launch has threads for in the sums' join (2^26) and, of rows, in both passes (2^30)."""
    def check(R, D, dx):
        g = torch.Generator(device="cuda").manual_seed(D)
        x, dy = (torch.empty(R, D, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
        mean, rstd = torch.full((R,), 0.125, device="cuda"), torch.full((R,), 0.5, device="cuda")
        got = L.layer_norm_backward(dy, x, mean, rstd, need_x=dx)
        for c in range(0, D, 1 << 26):  # columns c ..
            part = slice(c, min(D, c + (1 << 26)))
            h, d = (x[:, part].double() - 0.125) * 0.5, dy[:, part].double()
            for a, want, size in ((got.weight, (d * h).sum(0), (d * h).abs().sum(0)), (got.bias, d.sum(0), d.abs().sum(0))):
                assert ((a[part].double() - want).abs() <= (R + 8) * V * size).all()
        return got.x, x, dy
    D = (1 << 26) + 25
    dx, x, dy = check(2, D, True)
    X, DY = x.double(), dy.double()
    h = (X - 0.125) * 0.5
    s1, s2 = DY.mean(1, keepdim=True), (DY * h).mean(1, keepdim=True)
    want = 0.5 * (DY - s1 - h * s2)
    c = chain(D) * V  # of sums of random signs: some thousandth of the terms' size over its root
    e = 0.5 * (c * DY.abs().mean(1, keepdim=True) + h.abs() * (c * (DY * h).abs().mean(1, keepdim=True)) + 8 * V * (DY.abs() + h.abs()))
    assert ((dx.double() - want).abs() <= e + unit(BF16) * (want.abs() + e)).all()
    del dx, x, dy, X, DY, h, want, e
    check(1, (1 << 30) + 77, False)
