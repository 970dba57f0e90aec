"""group_norm_act, dropout_act and dense_act against plain 64-bit formulas.

Tolerances are elementwise bounds from the number formats: u32 = 2^-24 and
u16 = 2^-8 are the unit roundoffs of fp32 (24 significant bits) and bf16 (8).  A product of K terms is
summed in fp32 in steps of 16 terms at most, so its error is below
(K / 16 + 8) * 2 u32 * (|a| @ |b|); an activation has slope below 1.2 and
second derivative below 1.2; a stored bf16 value adds u16 of itself.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
ACTS = [None, "silu", "gelu", "relu"]


# ------------------------------------------------------------------ 64-bit formulas
def philox4x32_10(ctr, key):
    """Philox4x32-10 of the 2011 paper on numpy uint64 arrays holding 32-bit words."""
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, dtype=np.uint64) for v in ctr]
    k = [int(v) for v in key]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & mask, (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(rows, cols, rate, seed, offset):
    per_row = -(-cols // 8)
    n = np.arange(rows * per_row, dtype=np.uint64)
    words = philox4x32_10([n & np.uint64(0xFFFFFFFF), n >> np.uint64(32), np.full_like(n, offset & 0xFFFFFFFF),
                           np.full_like(n, offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([(words[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF) for j in range(8)], axis=1)
    keep = bits.reshape(rows, per_row * 8)[:, :cols] >= round(rate * 65536)
    return torch.from_numpy(np.ascontiguousarray(keep)).cuda()


def act64(u, act):
    if act == "silu":
        return u * torch.sigmoid(u)
    if act == "gelu":
        return torch.nn.functional.gelu(u, approximate="tanh")
    return torch.relu(u) if act == "relu" else u


def slope64(u, act):
    u = u.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(u, act).sum(), u)[0]


def factor(rate):
    d = round(rate * 65536)
    return 0.0 if d == 65536 else 65536 / (65536 - d)


def drop64(x, rate, keep):
    return x if keep is None else torch.where(keep, x * factor(rate), torch.zeros_like(x))


def assert_within(got, want, bound, what=""):
    got = got.double()
    assert got.shape == want.shape, what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond, worst " \
        f"{float(((got - want).abs() / bound.clamp(min=1e-300)).max()):.2f} of the bound"
    assert bool(torch.isfinite(got).all()) or not bool(torch.isfinite(want).all()), what


def stored(v, dtype):
    """Rounding of a result of magnitude v to dtype, with fp32 arithmetic before it."""
    return v.abs() * (U16 * 1.01 if dtype == torch.bfloat16 else 0.0) + 1e-30


# ------------------------------------------------------------------ dropout
def test_generator_known_answers():
    """The paper's published vectors."""
    def hexes(ctr, key):
        return [int(v[0]) for v in philox4x32_10([np.array([c]) for c in ctr], key)]
    assert hexes([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert hexes([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,rate", [((1, 1), 0.5), ((3, 7), 0.3), ((2, 5, 333), 0.25), ((37, 768), 0.1),
                                        ((4, 129, 64), 0.9), ((1, 100001), 0.02)])
@pytest.mark.parametrize("with_res", [False, True])
def test_dropout_act(cuda, dtype, act, shape, rate, with_res):
    from selectssm_b200 import dropout_act
    torch.manual_seed(1)
    x = torch.randn(shape, device=cuda).to(dtype).requires_grad_()
    res = torch.randn(shape, device=cuda).to(dtype).requires_grad_() if with_res else None
    seed, offset = 0x9ABCDEF012345678, (5 << 40) + 3
    y = dropout_act(x, rate, (seed, offset), activation=act, residual=res)
    dy = torch.randn(shape, device=cuda).to(dtype)
    y.backward(dy)
    keep = keep_mask(int(np.prod(shape[:-1])), shape[-1], rate, seed, offset).view(shape)
    u = drop64(x.detach().double(), rate, keep)
    want = act64(u, act) + (res.detach().double() if with_res else 0)
    slack = 16 * U32 * (u.abs() + (res.detach().double().abs() if with_res else 0))
    assert_within(y.detach(), want, slack + stored(want, dtype), "y")
    dx = drop64(dy.double() * slope64(u, act), rate, keep)
    assert_within(x.grad, dx, 32 * U32 * dy.double().abs() * factor(rate) * (1 + u.abs()) + stored(dx, dtype), "dx")
    assert bool((x.grad[~keep] == 0).all())
    if with_res:
        assert torch.equal(res.grad, dy)


@pytest.mark.parametrize("rate", [0.0, 1.0])
def test_dropout_of_nothing_and_of_everything(cuda, rate):
    from selectssm_b200 import dropout_act
    x = torch.randn(9, 40, device=cuda, requires_grad=True)
    y = dropout_act(x, rate, (1, 2))
    y.sum().backward()
    assert torch.equal(y, x if rate == 0 else torch.zeros_like(x))
    assert torch.equal(x.grad, torch.full_like(x, 1.0 - rate))


@pytest.mark.parametrize("cols", [64, 61])
@pytest.mark.parametrize("act", ACTS)
def test_dropped_infinities_and_nans_leave_no_trace(cuda, cols, act):
    from selectssm_b200 import dropout_act
    keep = keep_mask(20, cols, 0.5, 3, 0)
    clean = torch.randn(20, cols, device=cuda)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        x = torch.where(keep, clean, torch.full_like(clean, bad)).requires_grad_()
        y = dropout_act(x, 0.5, (3, 0), activation=act)
        y.sum().backward()
        ref = clean.clone().requires_grad_()
        yr = dropout_act(ref, 0.5, (3, 0), activation=act)
        yr.sum().backward()
        assert torch.equal(y, yr) and torch.equal(x.grad, ref.grad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropout_strided_rows_and_broadcast_residual(cuda, dtype):
    from selectssm_b200 import dropout_act
    torch.manual_seed(2)
    wide = torch.randn(6, 11, 200, device=cuda).to(dtype)
    rng = (7, 8)
    for lo, hi in ((0, 64), (8, 72), (3, 67), (1, 200)):   # aligned, 16-byte aligned, unaligned, odd width
        x = wide[..., lo:hi]
        res = torch.randn(hi - lo, device=cuda).to(dtype).requires_grad_()
        xd = x.contiguous().requires_grad_()
        xs = x.detach().requires_grad_()
        a = dropout_act(xs, 0.4, rng, activation="silu", residual=res)
        b = dropout_act(xd, 0.4, rng, activation="silu", residual=res.detach().expand(xd.shape).contiguous())
        assert torch.equal(a, b)
        dy = torch.randn(6, 11, 200, device=cuda).to(dtype)[..., lo:hi]
        ga, gr = torch.autograd.grad(a, (xs, res), dy)
        gb, = torch.autograd.grad(b, xd, dy.contiguous())
        assert torch.equal(ga, gb)
        assert_within(gr, dy.double().sum((0, 1)), 1e-5 + 66 * U16 * dy.double().abs().sum((0, 1)) / 8)


def test_dropout_mask_from_a_device_tensor_and_by_offset(cuda):
    from selectssm_b200 import dropout_act
    x = torch.ones(64, 96, device=cuda)
    rng = torch.tensor([-5, 9], dtype=torch.int64, device=cuda)
    a = dropout_act(x, 0.5, rng)
    assert torch.equal(a, dropout_act(x, 0.5, ((1 << 64) - 5, 9)))
    rng[1] = 10
    b = dropout_act(x, 0.5, rng)
    assert not torch.equal(a, b)
    kept = float((b != 0).float().mean())
    assert abs(kept - 0.5) < 5 * 0.5 / 64 / 96 ** 0.5 * 8 ** 0.5  # five standard deviations, generously


def test_dropout_beyond_32_bit_offsets(cuda):
    """Elements past 2^32: row and address arithmetic hold there."""
    from selectssm_b200 import dropout_act
    cols = 1 << 16
    rows = (1 << 16) + 3
    x = torch.ones(rows, cols, device=cuda, dtype=torch.bfloat16)
    y = dropout_act(x, 0.5, (11, 12))
    tail = y[-2:].float()
    del y
    n = 2 * cols // 8
    first = (rows - 2) * (cols // 8)
    idx = np.arange(first, first + n, dtype=np.uint64)
    w = philox4x32_10([idx & np.uint64(0xFFFFFFFF), idx >> np.uint64(32), np.full_like(idx, 12), np.zeros_like(idx)], (11, 0))
    bits = np.stack([(w[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF) for j in range(8)], axis=1)
    keep = torch.from_numpy((bits.reshape(2, cols) >= 32768).astype(np.float32)).cuda()
    assert torch.equal(tail, keep * 2)


# ------------------------------------------------------------------ group norm
def gn64(x, scale, bias, groups, eps, act, dy):
    B, D = x.shape[0], x.shape[-1]
    x3 = x.detach().double().reshape(B, -1, D)
    g = x3.view(B, -1, groups, D // groups)
    mu = g.mean((1, 3), keepdim=True)
    sd = ((g - mu).pow(2).mean((1, 3), keepdim=True) + eps).sqrt()
    xhat = ((g - mu) / sd).view_as(x3)
    u = xhat * scale + bias
    du = dy.double().view_as(x3) * slope64(u, act)
    gg = (du * scale).view_as(g)
    hg = xhat.view_as(g)
    dx = (gg - gg.mean((1, 3), keepdim=True) - hg * (gg * hg).mean((1, 3), keepdim=True)) / sd
    out = dict(y=act64(u, act), dx=dx.view_as(x3), dscale=(du * xhat).sum((0, 1)), dbias=du.sum((0, 1)))
    # xhat's error: rounding of x - mean, and a mean good to 16 u32 of the values it averages
    e = 16 * U32 * ((g.abs() + mu.abs()) / sd + hg.abs() + g.abs().mean((1, 3), keepdim=True) / sd).view_as(x3)
    ey = 1.2 * (e * scale.abs() + 8 * U32 * (u.abs() + 1))
    edu = dy.double().view_as(x3).abs() * (1.2 * (e * scale.abs() + 8 * U32 * (u.abs() + 1)) + 8 * U32)
    ex = (edu * scale.abs()).view_as(g)
    mean = lambda t: t.abs().mean((1, 3), keepdim=True)
    ev = e.view_as(g)
    edx = (ex + mean(ex) + ev * mean(gg * hg) + hg.abs() * (mean(ex * hg) + mean(gg * ev))
           + 32 * U32 * (gg.abs() + mean(gg) + hg.abs() * mean(gg * hg))) / sd
    n = x3.shape[0] * x3.shape[1]
    acc = (16 + n ** 0.5) * U32
    tol = dict(y=ey, dx=edx.view_as(x3), dscale=(edu * xhat.abs() + du.abs() * e).sum((0, 1)) + acc * (du * xhat).abs().sum((0, 1)),
               dbias=edu.sum((0, 1)) + acc * du.abs().sum((0, 1)))
    return out, tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((1, 1, 8), 2), ((2, 1, 768), 32), ((3, 7, 33), 11), ((64, 1, 96), 32),
                                          ((2, 1021, 330), 10), ((5, 300, 64), 64), ((1, 5000, 256), 32),
                                          ((2, 2048, 768), 32), ((3, 513, 24), 1), ((2, 40, 2056), 8), ((2, 3, 4, 40), 5),
                                          ((1, 30000, 8), 1), ((2, 9, 5003), 1)])
def test_group_norm_act(cuda, dtype, act, shape, groups):
    from selectssm_b200 import group_norm_act
    torch.manual_seed(3)
    D = shape[-1]
    x = (torch.randn(shape, device=cuda) * 1.5 + 2 * torch.randn(D, device=cuda)).to(dtype).requires_grad_()
    scale = (1 + 0.2 * torch.randn(D, device=cuda)).requires_grad_()
    bias = (0.3 * torch.randn(D, device=cuda)).requires_grad_()
    dy = torch.randn(shape, device=cuda).to(dtype)
    y = group_norm_act(x, scale, bias, groups=groups, activation=act)
    if act == "relu":  # at the kink the slope is either one's
        with torch.no_grad():
            u = group_norm_act(x, scale, bias, groups=groups).double()
            dy = torch.where(u.abs() < 1e-3, torch.zeros_like(dy), dy)
    y.backward(dy)
    want, tol = gn64(x, scale.detach().double(), bias.detach().double(), groups, 1e-6, act, dy)
    for name, got in (("y", y), ("dx", x.grad)):
        assert_within(got.detach().reshape(want[name].shape), want[name], tol[name] + stored(want[name], dtype), name)
    for name, got in (("dscale", scale.grad), ("dbias", bias.grad)):
        assert_within(got, want[name], tol[name] + 1e-30, name)


@pytest.mark.parametrize("shape", [(2, 4000, 64), (2, 100000, 16)])
def test_group_norm_with_a_large_mean_and_one_outlier(cuda, shape):
    """Means a thousand times the spread, and a first value far from the rest:
    sums of squares would lose every digit of the variance."""
    from selectssm_b200 import group_norm_act
    torch.manual_seed(4)
    x = 1000 + torch.randn(shape, device=cuda)
    x[:, 0, :] = 3000
    y = group_norm_act(x, groups=8)
    dy = torch.zeros(shape, device=cuda)
    one, zero = (torch.full((shape[-1],), v, device=cuda, dtype=torch.float64) for v in (1.0, 0.0))
    want, tol = gn64(x, one, zero, 8, 1e-6, None, dy)
    assert_within(y.reshape(want["y"].shape), want["y"], tol["y"] + 1e-30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_of_many_short_rows(cuda, dtype):
    """A norm per token: far more batch rows than clusters, each taking several."""
    from selectssm_b200 import group_norm_act
    torch.manual_seed(10)
    shape, groups = (70001, 1, 48), 6
    x = torch.randn(shape, device=cuda).to(dtype).requires_grad_()
    scale, bias = (t.requires_grad_() for t in (1 + 0.1 * torch.randn(48, device=cuda), torch.randn(48, device=cuda)))
    dy = torch.randn(shape, device=cuda).to(dtype)
    y = group_norm_act(x, scale, bias, groups=groups, activation="silu")
    y.backward(dy)
    want, tol = gn64(x, scale.detach().double(), bias.detach().double(), groups, 1e-6, "silu", dy)
    for name, got in (("y", y.detach()), ("dx", x.grad)):
        assert_within(got, want[name], tol[name] + stored(want[name], dtype), name)
    for name, got in (("dscale", scale.grad), ("dbias", bias.grad)):
        assert_within(got, want[name], tol[name] + 1e-30, name)


def test_group_norm_constant_input(cuda):
    """No spread: xhat is 0 and y the activated bias."""
    from selectssm_b200 import group_norm_act
    x = torch.full((2, 50, 64), 7.25, device=cuda, requires_grad=True)
    bias = torch.linspace(-1, 1, 64, device=cuda)
    y = group_norm_act(x, None, bias, groups=4, activation="silu")
    assert_within(y.detach(), act64(bias.double(), "silu").expand(2, 50, 64), torch.tensor(1e-6, device=cuda).double())
    y.sum().backward()
    assert bool(torch.isfinite(x.grad).all())


@pytest.mark.parametrize("op", ["norm", "dense"])
def test_gradients_agree_with_differences(cuda, op):
    """Directional differences of the forward in fp32: step 2^-7, so the
    truncation is about 2^-14 and the rounding about 2^-24 / 2^-7 = 2^-17 of a
    sum of 1e4 terms of both signs; 1% of the derivative's scale covers both."""
    from selectssm_b200 import dense_act, group_norm_act
    torch.manual_seed(5)
    if op == "norm":
        args = [torch.randn(3, 50, 64, device=cuda), 1 + 0.1 * torch.randn(64, device=cuda), torch.randn(64, device=cuda)]
        f = lambda a: group_norm_act(*a, groups=8, activation="silu")
    else:
        args = [torch.randn(150, 40, device=cuda), torch.randn(40, 64, device=cuda) / 6, torch.randn(64, device=cuda)]
        f = lambda a: dense_act(*a, activation="gelu", rate=0.25, rng=(1, 1))
    leaves = [a.clone().requires_grad_() for a in args]
    y = f(leaves)
    dy = torch.randn_like(y)
    grads = torch.autograd.grad(y, leaves, dy)
    h = 2.0 ** -7
    for i in range(3):
        v = torch.randn_like(args[i])
        ends = []
        for s in (h, -h):
            moved = list(args)
            moved[i] = args[i] + s * v
            ends.append((f(moved).double() * dy.double()).sum())
        numeric, formula = float((ends[0] - ends[1]) / (2 * h)), float((grads[i].double() * v.double()).sum())
        scale = float((grads[i].double().norm() * v.double().norm()) / v.numel() ** 0.5)
        assert abs(numeric - formula) < 0.01 * max(scale, abs(formula)), i


# ------------------------------------------------------------------ dense layer
def dense64(x, w, b, res, act, rate, keep, dy, dtype):
    x, w = x.detach().double(), w.detach().double()
    M, K = x.shape
    N = w.shape[1]
    steps = lambda k: (k / 16 + 8) * 2 * U32
    pre = x @ w + (0 if b is None else b.detach().double())
    epre = steps(K) * (x.abs() @ w.abs() + (0 if b is None else b.detach().double().abs()))
    f = factor(rate)
    u = drop64(pre, rate, keep)
    y = act64(u, act) + (0 if res is None else res.double())
    ey = 1.2 * f * epre + 16 * U32 * (u.abs() + (0 if res is None else res.double().abs()))
    out, tol = dict(y=y), dict(y=ey + stored(y, dtype))
    dpre = drop64(dy.double() * slope64(u, act), rate, keep)
    half = dtype == torch.bfloat16
    # the kept pre-activation and dpre are rounded to the operands' type
    edpre = f * dy.double().abs() * (1.2 * f * (epre + (U16 * pre.abs() if half and act else 0)) + 16 * U32 * (1 + u.abs()))
    op = edpre + (U16 * 1.01 * dpre.abs() if half else 0)
    for name, a, bb, ea, k in (("dx", dpre, w.T, op, N), ("dw", x.T, dpre, None, M)):
        out[name] = a @ bb
        e = ea @ bb.abs() if ea is not None else x.T.abs() @ op
        tol[name] = e + steps(k) * (a.abs() @ bb.abs()) + stored(out[name], dtype)
    out["db"] = dpre.sum(0)
    tol["db"] = edpre.sum(0) + (16 + M ** 0.5) * U32 * dpre.abs().sum(0) + stored(out["db"], dtype)
    return out, tol


DENSE_SIZES = [(1, 1, 1), (1, 768, 1536), (2, 515, 1001), (7, 64, 8), (16, 128, 64), (17, 96, 250), (129, 64, 129),
               (128, 256, 256), (300, 1000, 72), (1021, 100, 515), (2048, 512, 256), (5000, 40, 24), (33, 4099, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", DENSE_SIZES)
@pytest.mark.parametrize("act,rate,with_res", [(None, 0.0, False), ("silu", 0.1, False), (None, 0.3, True),
                                               ("gelu", 0.0, True), ("relu", 0.5, True)])
def test_dense_act(cuda, dtype, sizes, act, rate, with_res):
    from selectssm_b200 import dense_act
    M, K, N = sizes
    torch.manual_seed(6)
    x = torch.randn(M, K, device=cuda).to(dtype).requires_grad_()
    w = (torch.randn(K, N, device=cuda) / K ** 0.5).to(dtype).requires_grad_()
    b = torch.randn(N, device=cuda).to(dtype).requires_grad_()
    res = torch.randn(M, N, device=cuda).to(dtype) if with_res else None
    dy = torch.randn(M, N, device=cuda).to(dtype)
    seed, offset = 77, 5
    y = dense_act(x, w, b, activation=act, residual=res, rate=rate, rng=(seed, offset))
    keep = keep_mask(M, N, rate, seed, offset) if rate else None
    if act == "relu":  # at the kink the slope is either one's
        pre = x.detach().double() @ w.detach().double() + b.detach().double()
        dy = torch.where(pre.abs() < 1e-2, torch.zeros_like(dy), dy)
    y.backward(dy)
    want, tol = dense64(x, w, b, res, act, rate, keep, dy, dtype)
    for name, got in (("y", y.detach()), ("dx", x.grad), ("dw", w.grad), ("db", b.grad)):
        assert_within(got, want[name], tol[name], name)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dense_strides_batches_and_master_weights(cuda, dtype, rows):
    """Slices of a wider buffer, a transposed kernel, fp32 weights under bf16
    activations, and leading axes give what dense operands of one type give."""
    from selectssm_b200 import dense_act
    torch.manual_seed(7)
    wide = torch.randn(2, rows, 400, device=cuda).to(dtype)
    master = torch.randn(72, 96, device=cuda).t().contiguous().t().requires_grad_()
    bias = torch.randn(96, device=cuda)
    for lo in (0, 8, 5):
        x = wide[..., lo:lo + 72].detach().requires_grad_()
        dy = wide[..., 300 - lo:396 - lo]
        y = dense_act(x, master, bias, activation="silu", residual=wide[..., 100:196])
        gx, gw = torch.autograd.grad(y, (x, master), dy)
        xc, wc = x.detach().reshape(-1, 72).contiguous().requires_grad_(), master.detach().to(dtype).contiguous().requires_grad_()
        yc = dense_act(xc, wc, bias, activation="silu", residual=wide[..., 100:196].reshape(-1, 96).contiguous())
        hx, hw = torch.autograd.grad(yc, (xc, wc), dy.reshape(-1, 96).contiguous())
        assert torch.equal(y.reshape(-1, 96), yc) and torch.equal(gx.reshape(-1, 72), hx)
        assert gw.dtype == torch.float32 and torch.equal(gw.to(dtype), hw)


def test_dense_partial_gradients(cuda):
    from selectssm_b200 import dense_act
    torch.manual_seed(8)
    x, w, b = torch.randn(50, 48, device=cuda), torch.randn(48, 64, device=cuda), torch.randn(64, device=cuda)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    dy = torch.randn(50, 64, device=cuda)
    ref = torch.autograd.grad(dense_act(*full, activation="silu"), full, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].clone().requires_grad_()
        g, = torch.autograd.grad(dense_act(*args, activation="silu"), args[i], dy)
        assert torch.equal(g, ref[i])
    res = torch.randn(50, 64, device=cuda, requires_grad=True)
    g, = torch.autograd.grad(dense_act(x, w, b, activation="silu", residual=res), res, dy)
    assert torch.equal(g, dy)


def test_dense_dropped_infinities_leave_no_trace(cuda):
    from selectssm_b200 import dense_act
    keep = keep_mask(1, 256, 0.5, 3, 0)[0]
    x, w = torch.randn(1, 64, device=cuda), torch.randn(64, 256, device=cuda)
    b = torch.where(keep, torch.zeros(256, device=cuda), torch.full((256,), float("inf"), device=cuda))
    y = dense_act(x.clone().requires_grad_(), w, b, activation="silu", rate=0.5, rng=(3, 0))
    assert bool(torch.isfinite(y).all()) and bool((y[0][~keep] == 0).all())


@pytest.mark.parametrize("sizes", [(3, 96, 72), (200, 700, 130), (300, 96, 257), (700, 333, 64)])
def test_dense_fp32_infinities_and_the_largest_values(cuda, sizes):
    """An infinite operand makes what it makes in fp32 arithmetic, in each of the
    three products, and leaves the other rows and columns alone; values next to
    the type's largest keep fp32 accuracy."""
    from selectssm_b200 import dense_act
    M, K, N = sizes
    inf = float("inf")
    torch.manual_seed(12)
    x = torch.randn(M, K, device=cuda)
    w = torch.randn(K, N, device=cuda) / K ** 0.5
    dy = torch.randn(M, N, device=cuda)
    x[0, 5], x[1, K - 1], x[2, 17] = inf, -inf, 3.0e38
    w[5, 3] = 0.0  # infinity times nothing is NaN
    dy[1, 2] = inf
    dy[2] *= 0.125  # (products with 3e38 stay finite)
    x.requires_grad_(), w.requires_grad_()
    y = dense_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x64, w64, d64 = (t.detach().double() for t in (x, w, dy))
    for name, got, a, b in (("y", y.detach(), x64, w64), ("dx", dx, d64, w64.t()), ("dw", dw, x64.t(), d64)):
        want = (a @ b)
        clean = torch.isfinite(a).all(1)[:, None] & torch.isfinite(b).all(0)[None, :]
        # (inf * finite summed by hand: a 64-bit product may order its sums either way, its class is the same)
        assert torch.equal(torch.isnan(got)[~clean], torch.isnan(want)[~clean]), name
        odd = ~clean & ~torch.isnan(want)
        assert torch.equal(got[odd].double(), want[odd]), name
        # additions to the tensor core's accumulator are cut at 2^-23 of it, 32 in a row, and a
        # few roundings more; the planes leave 3 * 2^-24 of a product out
        bound = 40 * 2.0 ** -23 * (a.abs() @ b.abs())
        assert_within(got[clean], want[clean], bound[clean], name)


def test_dense_infinities_under_a_bf16_kernel(cuda):
    """The gradient of a bf16 kernel under fp32 activations is summed from the same planes."""
    from selectssm_b200 import dense_act
    torch.manual_seed(13)
    x = torch.randn(150, 72, device=cuda)
    x[4, 7] = float("inf")
    w = torch.randn(72, 96, device=cuda).bfloat16().requires_grad_()
    dy = torch.randn(150, 96, device=cuda).bfloat16().float()  # (whose lower planes are zeros)
    dw, = torch.autograd.grad(dense_act(x, w), w, dy)
    want = x.double().t() @ dy.double()
    assert dw.dtype == torch.bfloat16 and torch.equal(dw[7].double(), want[7])
    rest = [i for i in range(72) if i != 7]
    bound = 40 * 2.0 ** -23 * (x[:, rest].double().abs().t() @ dy.double().abs())
    assert_within(dw[rest], want[rest], bound + stored(want[rest], torch.bfloat16), "dw")


@pytest.mark.parametrize("sizes", [(129, 5000, 136), (2000, 520, 390), (513, 1032, 4200)])
def test_dense_fp32_over_long_sums(cuda, sizes):
    """Sums that pass through several accumulators, in whole and in cut K loops."""
    from selectssm_b200 import dense_act
    M, K, N = sizes
    torch.manual_seed(14)
    x = torch.rand(M, K, device=cuda).requires_grad_()  # of one sign: every addition is at the size of the result
    w = torch.rand(K, N, device=cuda).requires_grad_()
    dy = torch.rand(M, N, device=cuda)
    y = dense_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x64, w64, d64 = x.detach().double(), w.detach().double(), dy.double()
    for name, got, want in (("y", y.detach(), x64 @ w64), ("dx", dx, d64 @ w64.t()), ("dw", dw, x64.t() @ d64)):
        assert_within(got, want, 40 * 2.0 ** -23 * want, name)


def test_no_rows(cuda):
    from selectssm_b200 import dense_act, dropout_act, group_norm_act
    x = torch.empty(0, 16, device=cuda, requires_grad=True)
    w, b = torch.randn(16, 24, device=cuda, requires_grad=True), torch.randn(24, device=cuda, requires_grad=True)
    y = dense_act(x, w, b, activation="silu")
    assert y.shape == (0, 24)
    y.sum().backward()
    assert bool((w.grad == 0).all()) and bool((b.grad == 0).all()) and x.grad.shape == (0, 16)
    assert dropout_act(x, 0.5, (1, 1)).shape == (0, 16)
    s = torch.ones(16, device=cuda, requires_grad=True)
    for shape in ((0, 5, 16), (3, 0, 16)):
        z = group_norm_act(torch.empty(shape, device=cuda), s, groups=4)
        assert z.shape == shape
        g, = torch.autograd.grad(z.sum(), s)
        assert bool((g == 0).all())


# ------------------------------------------------------------------ as a program uses them
def _mlp_half(x, p, rng):
    from selectssm_b200 import dense_act, dropout_act, group_norm_act
    h = group_norm_act(x, p["scale"], p["bias"], groups=8, activation="silu")
    h = dense_act(h, p["w1"], p["b1"], activation="silu", rate=0.1, rng=rng)
    h = dropout_act(h, 0.2, rng)
    return dense_act(h, p["w2"], p["b2"], residual=x, rate=0.1, rng=rng)


def _mlp_params(cuda):
    torch.manual_seed(9)
    n = lambda *s: torch.randn(*s, device=cuda)
    return {k: v.requires_grad_() for k, v in dict(scale=1 + 0.1 * n(64), bias=0.1 * n(64), w1=n(64, 128) / 8, b1=n(128),
                                                   w2=n(128, 64) / 11, b2=n(64)).items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeated_and_other_stream_calls_are_bit_identical(cuda, dtype):
    p = _mlp_params(cuda)
    x = torch.randn(4, 700, 64, device=cuda).to(dtype).requires_grad_()
    runs = []
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side, torch.cuda.current_stream()):
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            y = _mlp_half(x, p, (1, 2))
            runs.append([y, *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))])
        torch.cuda.default_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_captured_step_follows_the_device_rng(cuda):
    p = _mlp_params(cuda)
    x = torch.randn(2, 300, 64, device=cuda, requires_grad=True)
    rng = torch.tensor([4, 0], dtype=torch.int64, device=cuda)

    def step():
        y = _mlp_half(x, p, rng)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for offset in (5, 6):
        rng[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("shape,groups", [((3, 50, 64), 8), ((1, 60000, 32), 2)])
def test_group_norm_with_and_without_statistics(cuda, shape, groups):
    """A call that records no gradient keeps no statistics, in either form, and gives the same bits."""
    from selectssm_b200 import group_norm_act
    torch.manual_seed(15)
    x = torch.randn(shape, device=cuda)
    y = group_norm_act(x, groups=groups, activation="silu")
    assert torch.equal(y, group_norm_act(x.clone().requires_grad_(), groups=groups, activation="silu"))


def test_dense_fp32_sums_that_start_the_small_products_afresh(cuda):
    """More tiles than CTAs, so that the K loop stays whole, and more than 4096 of K."""
    from selectssm_b200 import dense_act
    torch.manual_seed(16)
    x, w = torch.rand(1530, 4700, device=cuda), torch.rand(4700, 1660, device=cuda)
    want = x.double() @ w.double()
    # a sum of one sign grows from nothing, so its additions are cut at half of 2^-23 of the result
    # on average: 16 of the leading products, 3 of the small ones, 5 of ten cuts joined in fp32
    assert_within(dense_act(x, w), want, 25 * 2.0 ** -23 * want, "y")


@pytest.mark.parametrize("which", ["x", "scale", "kernel", "bias", "residual"])
def test_forward_mode_tangents_are_refused(cuda, which):
    from torch.autograd import forward_ad
    from selectssm_b200 import dense_act, dropout_act, group_norm_act
    a = dict(x=torch.randn(20, 5, 16, device=cuda), scale=torch.ones(16, device=cuda), kernel=torch.randn(16, 16, device=cuda),
             bias=torch.zeros(16, device=cuda), residual=torch.zeros(20, 5, 16, device=cuda))
    calls = [("x residual", lambda p: dropout_act(p["x"], 0.5, (1, 2), residual=p["residual"])),
             ("x scale bias", lambda p: group_norm_act(p["x"], p["scale"], p["bias"], groups=4)),
             ("x kernel bias residual", lambda p: dense_act(p["x"], p["kernel"], p["bias"], residual=p["residual"]))]
    for names, call in calls:
        with forward_ad.dual_level():
            p = dict(a)
            p[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    if which in names.split():
                        with pytest.raises(NotImplementedError):
                            call(p)
                    else:
                        call(p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((3, 50, 64), 8), ((1, 60000, 32), 2), ((4, 1, 96), 32)])
def test_group_norm_of_operands_at_any_address(cuda, dtype, shape, groups):
    """Contiguous views into a flat buffer, of x and (by the gradient of a concatenation) of dy."""
    from selectssm_b200 import group_norm_act
    torch.manual_seed(17)
    n = int(np.prod(shape))
    flat = torch.randn(n + 3, device=cuda).to(dtype)
    dy = torch.randn(n + 3, device=cuda).to(dtype)
    x = flat[3:].view(shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    runs = []
    for xi, di in ((x.detach().requires_grad_(), dy), (x.clone().requires_grad_(), dy)):
        y = group_norm_act(xi, groups=groups, activation="silu")
        runs.append((y.detach(), *torch.autograd.grad(torch.cat([y.new_zeros(3), y.flatten()]), xi, di)))
    xa = x.clone().requires_grad_()
    ya = group_norm_act(xa, groups=groups, activation="silu")
    runs.append((ya.detach(), *torch.autograd.grad(ya, xa, dy[3:].clone().view(shape))))
    for other in runs[:2]:
        assert all(torch.equal(a, b) for a, b in zip(runs[2], other))
    assert torch.equal(group_norm_act(x, groups=groups), group_norm_act(x.clone(), groups=groups))


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 61])
def test_dropout_relu_passes_nan_on(cuda, dtype, cols):
    """What is NaN where it is kept stays NaN, and its gradient is what torch's relu gives there."""
    from selectssm_b200 import dropout_act
    torch.manual_seed(18)
    x = torch.randn(20, cols, device=cuda).to(dtype)
    x[3, 5] = x[7, cols - 1] = x[19, 0] = float("nan")
    x[4, 4], x[4, 5] = float("inf"), -float("inf")
    dy = torch.randn(20, cols, device=cuda).to(dtype)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = dropout_act(a, 0.0, None, activation="relu"), torch.relu(b)
    ga, gb = torch.autograd.grad(ya, a, dy)[0], torch.autograd.grad(yb, b, dy)[0]
    assert _same(ya, yb) and _same(ga, gb)
    keep = keep_mask(20, cols, 0.5, 6, 1)
    y = dropout_act(x, 0.5, (6, 1), activation="relu")
    assert torch.equal(torch.isnan(y), torch.isnan(x) & keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 9, 200])
def test_dense_relu_passes_nan_on(cuda, dtype, rows):
    from selectssm_b200 import dense_act
    torch.manual_seed(19)
    x, w = torch.randn(rows, 72, device=cuda).to(dtype), torch.randn(72, 40, device=cuda).to(dtype)
    x[rows // 2, 7] = float("nan")
    y = dense_act(x, w, activation="relu")
    assert bool(torch.isnan(y[rows // 2]).all())
    rest = [r for r in range(rows) if r != rows // 2]
    assert bool(torch.isfinite(y[rest]).all()) and bool((y[rest] >= 0).all())
    # torch's relu lets the gradient of a NaN through
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(dense_act(xg, w, activation="relu"), xg, torch.ones_like(y))
    want, = torch.autograd.grad(torch.relu(xg @ w), xg, torch.ones_like(y))
    assert torch.equal(torch.isnan(g), torch.isnan(want))


@pytest.mark.parametrize("shape,groups", [((2, 50, 64), 8), ((1, 60000, 32), 2), ((6, 1, 33), 11)])
def test_group_norm_relu_passes_nan_on(cuda, shape, groups):
    from selectssm_b200 import group_norm_act
    x = torch.randn(shape, device=cuda)
    x[0, -1, 5] = float("nan")
    y = group_norm_act(x, groups=groups, activation="relu")
    cg = shape[-1] // groups
    hit = torch.zeros(shape, dtype=torch.bool, device=cuda)
    hit[0, :, 5 // cg * cg:(5 // cg + 1) * cg] = True
    assert torch.equal(torch.isnan(y), hit)


@pytest.mark.parametrize("op", ["dense", "norm"])
def test_threads_with_different_shapes(cuda, op):
    """Launches of one kernel with different amounts of shared memory, from two host threads
    at once: the C entries' calls alone, so that they overlap."""
    import ctypes
    import sys
    import threading
    from selectssm_b200 import _lib
    torch.manual_seed(20)
    lib, calls = _lib.load(), []
    stream = torch.cuda.current_stream().cuda_stream
    if op == "dense":  # 16 rows of fin / 8 values: 128 and 32 KB of shared memory
        w = torch.randn(16384, 512, device=cuda)
        for fin in (16384, 4096):
            x, y = torch.randn(16, fin, device=cuda), torch.empty(16, 512, device=cuda)
            p = _lib.SSMDenseParams()
            p.rows, p.fin, p.fout = 16, fin, 512
            p.x, p.kernel, p.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
            calls.append((lib.ssm_dense_act_fwd, p, x, y))
    else:  # a batch row a CTA: 70 and 50 KB
        for length in (260, 190):
            x = torch.randn(512, length, 64, device=cuda)
            y = torch.empty_like(x)
            p = _lib.SSMGroupNormParams()
            p.batch, p.seqlen, p.dim, p.groups, p.eps = 512, length, 64, 1, 1e-6
            p.x, p.y = x.data_ptr(), y.data_ptr()
            calls.append((lib.ssm_group_norm_act_fwd, p, x, y))
    codes = [set(), set()]

    def work(i):
        f, p = calls[i][:2]
        ref = ctypes.byref(p)
        for _ in range(20000):
            codes[i].add(f(ref, stream))

    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(before)
    torch.cuda.synchronize()
    assert codes == [{_lib.SSM_OK}, {_lib.SSM_OK}]


def _classes_agree(got, want, what=""):
    """NaN where want is NaN, the same infinity where it is infinite."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = torch.isinf(want)
    assert torch.equal(got[odd].double(), want[odd]) and not bool(torch.isinf(got[~odd]).any()), what


def test_dense_infinities_over_a_long_whole_sum(cuda):
    """More tiles than CTAs, so that a kernel's gradient is summed over all rows by one CTA
    each: with one infinity the other rows and columns keep their bits; with an infinite row,
    which reaches every sum, each is infinite or NaN as its terms say; a NaN row is NaN throughout."""
    from selectssm_b200 import dense_act
    torch.manual_seed(21)
    rows, fin, fout = 20011, 2056, 2000
    x, dy = torch.randn(rows, fin, device=cuda), torch.randn(rows, fout, device=cuda)
    w = torch.zeros(fin, fout, device=cuda, requires_grad=True)

    def dw(x, dy):
        return torch.autograd.grad(dense_act(x, w), w, dy)[0]

    clean = dw(x, dy)
    one = dy.clone()
    one[19000, 7] = float("inf")
    g = dw(x, one)
    assert torch.equal(g[:, 7], torch.sign(x[19000]) * float("inf"))
    rest = torch.arange(fout, device=cuda) != 7
    assert torch.equal(g[:, rest], clean[:, rest])
    dy[19990] = float("inf")
    dy[5, 3] = -float("inf")
    _classes_agree(dw(x, dy), x.double().t() @ dy.double())
    dy[40] = float("nan")
    assert bool(torch.isnan(dw(x, dy)).all())


@pytest.mark.parametrize("sizes", [(300, 96, 257), (129, 5000, 136), (20000, 72, 40)])
@pytest.mark.parametrize("act", ACTS)
def test_dense_fp32_infinities_through_the_epilogue(cuda, sizes, act):
    """Sums made again pass through bias, dropout, activation and residual like the others,
    with and without `pre` kept; what no infinity reaches keeps its bits."""
    from selectssm_b200 import dense_act
    M, K, N = sizes
    torch.manual_seed(22)
    x, w = torch.randn(M, K, device=cuda), torch.randn(K, N, device=cuda) / K ** 0.5
    b, res = torch.randn(N, device=cuda), torch.randn(M, N, device=cuda)
    call = lambda x, w: dense_act(x, w, b, activation=act, residual=res, rate=0.3, rng=(8, 9))
    clean = call(x, w)
    x[2, 17], x[M - 1, K - 1], x[9, 0] = float("inf"), -float("inf"), 3.0e38
    w[3, N - 1] = float("inf")
    w[0, 5] = 1.0e6  # a product of finite values beyond the largest
    keep = keep_mask(M, N, 0.3, 8, 9)
    pre = x.double() @ w.double() + b.double()
    u = drop64(torch.where(pre.abs() > 3.5e38, pre * float("inf"), pre), 0.3, keep)
    want = act64(u, act) + res.double()
    for y in (call(x, w), call(x.clone().requires_grad_(), w).detach()):
        hit = torch.zeros(M, N, dtype=torch.bool, device=cuda)
        hit[[2, 9, M - 1]] = True
        hit[:, [5, N - 1]] = True
        assert torch.equal(y[~hit], clean[~hit])
        sure = hit & ~((u.abs() > 1e30) & torch.isfinite(u))  # (a sum next to the largest value may pass it)
        _classes_agree(y[sure], want[sure])


# Sizes of which the product kernels make pairs of CTAs, several tiles a CTA (or pair) in a row, and
# cut K loops in bf16, all with ragged edges (tiles are 128 x 128 a CTA, of 148, or 256 x 256 a pair, of 74):
#   20001 x 1536 -> 776   y: pairs, 4.3 tiles each, last column tile 8 wide; dx: pairs, 6.4; dW: pairs, K in 3 parts
#   16500 x 264 -> 1000   y: pairs, 3.5; dx: single CTAs, 2.6; dW: single, K in 6 parts
#   20001 x 1031 -> 777   y and dx: pairs, rows that start anywhere; dW: single, K in 2 parts
#   40000 x 304 -> 304    y and dx: single CTAs, 6.3 tiles each; dW: K in 16 parts
#   768 x 32000 -> 1536   y: pairs, K in 4 parts joined with the epilogue; dx: pairs, 5.1; dW: pairs, 10.1
@pytest.mark.parametrize("sizes,act,rate,res_stride", [
    ((20001, 1536, 776), None, 0.1, 776), ((20001, 1536, 776), "silu", 0.0, 779), ((16500, 264, 1000), "silu", 0.1, None),
    ((20001, 1031, 777), "gelu", 0.3, 777), ((40000, 304, 304), None, 0.2, 312), ((768, 32000, 1536), "silu", 0.1, 1536)])
def test_dense_bf16_of_many_tiles(cuda, sizes, act, rate, res_stride):
    from selectssm_b200 import dense_act
    M, K, N = sizes
    dtype = torch.bfloat16
    torch.manual_seed(23)
    x = torch.randn(M, K, device=cuda).to(dtype).requires_grad_()
    w = (torch.randn(K, N, device=cuda) / K ** 0.5).to(dtype).requires_grad_()
    b = torch.randn(N, device=cuda).to(dtype).requires_grad_()
    res = torch.randn(M, res_stride, device=cuda).to(dtype)[:, :N] if res_stride else None
    dy = torch.randn(M, N, device=cuda).to(dtype)
    keep = keep_mask(M, N, rate, 31, 7) if rate else None
    runs = []
    for _ in range(2):
        y = dense_act(x, w, b, activation=act, residual=res, rate=rate, rng=(31, 7))
        runs.append((y.detach(), *torch.autograd.grad(y, (x, w, b), dy)))
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    want, tol = dense64(x, w, b, res, act, rate, keep, dy, dtype)
    for name, got in zip(("y", "dx", "dw", "db"), runs[0]):
        assert_within(got, want[name], tol[name], name)


def _needs(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB of the GPU's memory")


def test_dense_counters_beyond_32_bits(cuda):
    """Three dropout counters a row, more than 2^32 of them, and 24e9 outputs."""
    from selectssm_b200 import dense_act
    torch.cuda.empty_cache()
    _needs(90)
    torch.manual_seed(24)
    rows, fin, fout, tail = (1 << 32) // 3 + 60, 8, 17, 100
    x = torch.zeros(rows, fin, device=cuda, dtype=torch.bfloat16)
    x[-tail:] = torch.randn(tail, fin, device=cuda).bfloat16()
    w, b = torch.randn(fin, fout, device=cuda).bfloat16(), torch.randn(fout, device=cuda).bfloat16()
    y = dense_act(x, w, b, rate=0.5, rng=(11, 12))[-tail:].double()
    idx = np.arange((rows - tail) * 3, rows * 3, dtype=np.uint64)
    assert idx[0] < 1 << 32 < idx[-1]
    c = philox4x32_10([idx & np.uint64(0xFFFFFFFF), idx >> np.uint64(32), np.full_like(idx, 12), np.zeros_like(idx)], (11, 0))
    bits = np.stack([(c[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF) for j in range(8)], axis=1)
    keep = torch.from_numpy(np.ascontiguousarray(bits.reshape(tail, 24)[:, :fout] >= 32768)).to(cuda)
    want = drop64(x[-tail:].double() @ w.double() + b.double(), 0.5, keep)
    assert_within(y, want, 32 * U32 * (x[-tail:].double().abs() @ w.double().abs() + b.double().abs()) + stored(want, torch.bfloat16))
    del x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape,groups", [((3, 1500001, 512), 64), ((70000001, 1, 32), 4)])
def test_group_norm_beyond_32_bit_offsets(cuda, shape, groups):
    """More than 2^31 elements, in the split and in the held form: the last channels' group of the last rows."""
    from selectssm_b200 import group_norm_act
    torch.cuda.empty_cache()
    _needs(60)
    torch.manual_seed(25)
    B, L, D = shape
    cg = D // groups
    x = torch.empty(shape, device=cuda, dtype=torch.bfloat16).normal_().requires_grad_()
    dy = torch.empty(shape, device=cuda, dtype=torch.bfloat16).normal_()
    scale, bias = 1 + 0.2 * torch.randn(D, device=cuda), 0.3 * torch.randn(D, device=cuda)
    y = group_norm_act(x, scale, bias, groups=groups, activation="silu")
    dx, = torch.autograd.grad(y, x, dy)
    last = (slice(-2, None), slice(None), slice(-cg, None))
    want, tol = gn64(x[last], scale[-cg:].double(), bias[-cg:].double(), 1, 1e-6, "silu", dy[last].contiguous())
    for name, got in (("y", y), ("dx", dx)):
        got = got.detach()[last]
        assert_within(got, want[name], tol[name] + stored(want[name], torch.bfloat16), name)
    del x, y, dx, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(17, 1, 1), (33, 3, 1), (1000, 128, 1), (17, 1, 300), (50, 2, 7), (20000, 1, 9)])
@pytest.mark.parametrize("wide", [False, True])
def test_dense_smallest_widths(cuda, dtype, sizes, wide):
    """One column in or out past the few-row form, from rows of their own and from slices TMA can address."""
    from selectssm_b200 import dense_act
    M, K, N = sizes
    torch.manual_seed(26)
    x = torch.randn(M, (K + 15) // 8 * 8 if wide else K, device=cuda).to(dtype)[:, :K].requires_grad_()
    w, b = torch.randn(K, N, device=cuda).to(dtype).requires_grad_(), torch.randn(N, device=cuda).to(dtype).requires_grad_()
    dy = torch.randn(M, 24 if wide else N, device=cuda).to(dtype)[:, :N] if N < 24 else torch.randn(M, N, device=cuda).to(dtype)
    for act, rate in (("silu", 0.25), (None, 0.0)):
        keep = keep_mask(M, N, rate, 2, 3) if rate else None
        y = dense_act(x, w, b, activation=act, rate=rate, rng=(2, 3))
        grads = torch.autograd.grad(y, (x, w, b), dy)
        want, tol = dense64(x, w, b, None, act, rate, keep, dy, dtype)
        for name, got in zip(("y", "dx", "dw", "db"), (y.detach(), *grads)):
            assert_within(got, want[name], tol[name], name)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dense_with_everything_dropped(cuda, dtype, rows):
    from selectssm_b200 import dense_act
    x, w = torch.randn(rows, 40, device=cuda).to(dtype), torch.randn(40, 24, device=cuda).to(dtype)
    x[1, 1] = float("inf")
    x.requires_grad_(), w.requires_grad_()
    res = torch.randn(rows, 24, device=cuda).to(dtype)
    y = dense_act(x, w, activation="silu", residual=res, rate=1.0, rng=(1, 1))
    assert torch.equal(y, res)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool((dx == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((2, 50, 1), 1), ((5, 1, 1), 1), ((3, 1, 2), 2), ((1, 200001, 1), 1), ((2, 1), 1)])
def test_group_norm_smallest_widths(cuda, dtype, shape, groups):
    from selectssm_b200 import group_norm_act
    torch.manual_seed(27)
    D = shape[-1]
    x = torch.randn(shape, device=cuda).to(dtype).requires_grad_()
    scale, bias = torch.randn(D, device=cuda).requires_grad_(), torch.randn(D, device=cuda).requires_grad_()
    dy = torch.randn(shape, device=cuda).to(dtype)
    y = group_norm_act(x, scale, bias, groups=groups, activation="gelu")
    y.backward(dy)
    want, tol = gn64(x, scale.detach().double(), bias.detach().double(), groups, 1e-6, "gelu", dy)
    for name, got in (("y", y.detach()), ("dx", x.grad)):
        assert_within(got.reshape(want[name].shape), want[name], tol[name] + stored(want[name], dtype), name)
    for name, got in (("dscale", scale.grad), ("dbias", bias.grad)):
        assert_within(got, want[name], tol[name] + 1e-30, name)
