"""Linear with its epilogue, LayerNormalization, TokenLogProbs and the gradients against plain formulas in 64 bits.

Tolerances.  u is the unit roundoff of the output's type (half of torch.finfo.eps): the one rounding of a result.  A sum of n terms in 32
bits is off by at most n 2^-23 times the sum of the terms' magnitudes, whatever its order and whether the additions round or truncate.  An
elementary function is taken as good to 2^-20 relative (a few ulp of its 32-bit value and of its argument)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "Relu", "Gelu", "GeluTanh", "Swish", "Sigmoid", "Tanh"]
E32, EF = 2.0 ** -23, 2.0 ** -20


def _u(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps  # the spacing of subnormal values


def _act64(z, act):
    return {None: lambda: z, "Relu": lambda: z.clamp(min=0), "Gelu": lambda: 0.5 * z * torch.special.erfc(-z / math.sqrt(2)),
            "GeluTanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)), "Swish": lambda: z * torch.sigmoid(z),
            "Sigmoid": lambda: torch.sigmoid(z), "Tanh": lambda: torch.tanh(z)}[act]()


def _check(got, want, bound, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    same = (got == want) | torch.isnan(want)
    over = ((got - want).abs() > bound) & ~same
    assert not over.any(), "%s: %d of %d off, worst %.3g of its bound" % (what, int(over.sum()), over.numel(), float(((got - want).abs() / bound)[over].max()))


def _linear64(x, w, b, act, r, first):
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    if r is not None and first:
        z, mag = z + r.double(), mag + r.double().abs()
    y = _act64(z, act)
    # the activations' slopes are at most 1.13; their own error is relative to the larger of argument and value (Sigmoid, Tanh: at most 1)
    err = 1.2 * (x.shape[-1] + 4) * E32 * mag + EF * torch.maximum(y.abs(), (y if act is None else torch.minimum(z.abs(), torch.ones_like(z))).abs())
    if r is not None and not first:
        err = err + E32 * (y.abs() + r.double().abs())
        y = y + r.double()
    return y, err + _u(x.dtype) * 1.001 * y.abs() + _tiny(x.dtype)


def _check_linear(ops, dev, m, k, o, dtype, act, residual, bias=True, bias32=False, seed=0, pitch=0):
    g = torch.Generator(device=dev).manual_seed(seed + m * 7 + k * 3 + o)
    x = torch.randn((m, k + pitch), device=dev, generator=g).to(dtype)[:, :k]
    w = (torch.randn((o, k + pitch), device=dev, generator=g) / math.sqrt(max(k, 1))).to(dtype)[:, :k]
    b = torch.randn(o, device=dev, generator=g).to(torch.float32 if bias32 else dtype) if bias else None
    r = torch.randn((m, o + pitch), device=dev, generator=g).to(dtype)[:, :o] if residual else None
    y = ops.Linear(x, w, b, activation=act, residual=r, residual_first=residual == "first")
    assert y.shape == (m, o) and y.dtype == dtype and y.is_contiguous()
    want, bound = _linear64(x, w, b, act, r, residual == "first")
    _check(y, want, bound, "Linear %s" % ((m, k, o, dtype, act, residual),))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("residual", [None, "last", "first"])
@pytest.mark.parametrize("m,k,o", [(37, 96, 72), (20, 96, 2500), (140, 96, 600), (1100, 64, 2048)])  # one for each kernel
def test_linear_epilogues(ops, dev, dtype, act, residual, m, k, o):
    _check_linear(ops, dev, m, k, o, dtype, act, residual, bias32=residual is None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,o", [(1, 1, 1), (1, 0, 5), (3, 8, 1), (1, 512, 4096), (2, 2048, 1000), (16, 64, 16), (17, 200, 33), (33, 1283, 129), (128, 128, 128), (129, 72, 257),
                                   (3, 4096, 5000), (9, 200, 3001), (20, 333, 2500), (40, 1283, 1999), (64, 8, 5000), (61, 8192, 1300),
                                   (256, 2048, 1000), (300, 33, 511), (509, 1283, 997), (1024, 512, 768), (777, 4096, 640), (2500, 264, 1500)])
def test_linear_extents(ops, dev, dtype, m, k, o):
    _check_linear(ops, dev, m, k, o, dtype, "Gelu", "last" if o % 2 else "first", bias=m != 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [1, 8, 24])
@pytest.mark.parametrize("m", [1, 40, 700])
def test_linear_rows_of_wider_buffers(ops, dev, dtype, pitch, m):
    _check_linear(ops, dev, m, 320, 264, dtype, "Swish", "last", pitch=pitch)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", list(range(1, 10)) + [16, 25, 400])
@pytest.mark.parametrize("k,o,pitch", [(4100, 5, 0), (1023, 131, 0), (70, 2050, 1), (3, 64, 4), (6948, 26, 0), (2047, 700, 5), (64, 30, 8)])
def test_linear_few_outputs(ops, dev, dtype, m, k, o, pitch):
    _check_linear(ops, dev, m, k, o, dtype, "Tanh", "first" if m % 2 else "last", pitch=pitch)


@pytest.mark.parametrize("m,k,o", [(2048, 64, 2000), (1900, 17, 2100), (349, 500, 3125), (1024, 33, 1000), (300, 40, 5000), (65, 300, 20000), (2200000, 3, 2)])
def test_linear_fp32_without_an_epilogue_is_one_chain(ops, dev, m, k, o):
    """y = b + a chain of fused multiply-adds in ascending k, in large products as in small ones: sampled outputs, bit for bit."""
    g = torch.Generator(device=dev).manual_seed(m + k + o)
    x, w, b = torch.randn((m, k), device=dev, generator=g), torch.randn((o, k), device=dev, generator=g), torch.randn(o, device=dev, generator=g)
    y = ops.Linear(x, w, b)
    rows = torch.cat([torch.tensor([0, m - 1, m // 2], device=dev), torch.randint(0, m, (29,), device=dev, generator=g)])
    cols = torch.cat([torch.tensor([0, o - 1], device=dev), torch.randint(0, o, (30,), device=dev, generator=g)])
    got = y[rows][:, cols].cpu()
    xs, ws = x[rows].cpu(), w[cols].cpu()
    acc = torch.zeros((32, 32))
    for i in range(k):  # (a product of two fp32 values is exact in 64 bits; its sum rounds to 64 and then to 32, which is one rounding but next to a tie)
        acc = (xs[:, i:i + 1].double() * ws[:, i].double() + acc.double()).float()
    want = acc + b[cols].cpu()
    assert torch.equal(got, ops.Linear(x[rows], w[cols], b[cols]).cpu())  # another kernel
    # a tie decided the other way moves a chain by a unit in the last place of its value then
    mag = xs.double().abs() @ ws.double().abs().t() + b[cols].cpu().double().abs()
    assert (got == want).float().mean() > 0.99 and ((got.double() - want.double()).abs() <= k * E32 * mag).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_offset_addresses_and_other_strides(ops, dev, dtype):
    """Operands that start off a 16-byte boundary, a transposed weight, rows that overlap (an expanded one), a batch of leading dimensions."""
    g = torch.Generator(device=dev).manual_seed(5)
    buf = torch.randn(64 * 128 + 200 * 128 + 64 * 200 + 9, device=dev, generator=g).to(dtype)
    x, w, r = buf[1:1 + 64 * 128].view(64, 128), buf[3 + 64 * 128:][:200 * 128].view(200, 128), buf[5 + 264 * 128:][:64 * 200].view(64, 200)
    want, bound = _linear64(x, w, None, "Relu", r, False)
    _check(ops.Linear(x, w, activation="Relu", residual=r), want, bound)
    wt = w.t().contiguous().t()
    _check(ops.Linear(x, wt, activation="Relu", residual=r), want, bound)
    xe = x[:1].expand(64, 128)
    want, bound = _linear64(xe, w, None, None, r, False)
    _check(ops.Linear(xe, w, residual=r), want, bound)
    x4 = x.view(2, 4, 8, 128)
    want, bound = _linear64(x, w, None, "Tanh", None, False)
    y4 = ops.Linear(x4, w, activation="Tanh")
    assert y4.shape == (2, 4, 8, 200)
    _check(y4.view(64, 200), want, bound)
    xp = x4.permute(1, 0, 2, 3)
    assert torch.equal(ops.Linear(xp, w, activation="Tanh"), y4.permute(1, 0, 2, 3))


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_a_vector(ops, dev, dtype):
    g = torch.Generator(device=dev).manual_seed(8)
    x, w, r = (torch.randn(s, device=dev, generator=g).to(dtype) for s in ((70,), (33, 70), (33,)))
    want, bound = _linear64(x[None], w, None, "Tanh", r[None], True)
    y = ops.Linear(x, w, activation="Tanh", residual=r, residual_first=True)
    assert y.shape == (33,)
    _check(y[None], want, bound)
    wide = w[:1].expand(33, 70)  # rows that overlap
    want, bound = _linear64(x[None], wide, None, None, r[None], False)
    _check(ops.Linear(x, wide, residual=r)[None], want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_without_sums_or_outputs(ops, dev, dtype):
    z = lambda *s: torch.zeros(s, dtype=dtype, device=dev)  # noqa: E731
    assert ops.Linear(z(0, 8), z(5, 8), activation="Relu").shape == (0, 5)
    assert ops.Linear(z(4, 8), z(0, 8)).shape == (4, 0) and ops.Linear(z(2, 0, 8), z(5, 8)).shape == (2, 0, 5)
    b = torch.tensor([-1.0, 2.0, 0.5], dtype=dtype, device=dev)
    assert torch.equal(ops.Linear(z(2, 0), z(3, 0), b, activation="Relu"), torch.clamp(b, min=0).expand(2, 3))


def test_linear_special_values(ops, dev):
    """NaN and infinities travel as the formula has them; an activation of a large negative value is zero, not NaN."""
    for dtype in TYPES:
        for m, o in ((1, 16), (200, 16), (20, 2500), (200, 1100), (1100, 2048)):
            x = torch.zeros((m, 64), dtype=dtype, device=dev)
            w = torch.zeros((o, 64), dtype=dtype, device=dev)
            w[:, 0] = 1
            x[:, 0] = torch.tensor([float("nan"), float("inf"), -300.0, 300.0], dtype=dtype, device=dev)[torch.arange(m, device=dev) % 4]
            for act in ACTS:
                y = ops.Linear(x, w, activation=act, residual=torch.zeros((m, o), dtype=dtype, device=dev)).float()
                assert torch.isnan(y[0]).all(), act
                if m > 1:
                    assert torch.equal(y[1], torch.full_like(y[1], 1.0 if act in ("Sigmoid", "Tanh") else float("inf"))), act
                    assert torch.equal(y[2], torch.full_like(y[2], {None: -300.0, "Tanh": -1.0}.get(act, 0.0))), act
                    assert torch.equal(y[3], torch.full_like(y[3], 1.0 if act in ("Sigmoid", "Tanh") else 300.0)), act


def test_linear_refusals(ops, dev):
    x, w = torch.zeros((4, 8), dtype=torch.bfloat16, device=dev), torch.zeros((3, 8), dtype=torch.bfloat16, device=dev)
    bad = [lambda: ops.Linear(x, w.half()), lambda: ops.Linear(x, w[:, :7]), lambda: ops.Linear(x, w[0]), lambda: ops.Linear(x.double(), w.double()),
           lambda: ops.Linear(x, w, torch.zeros(4, device=dev)), lambda: ops.Linear(x, w, torch.zeros(3, dtype=torch.float16, device=dev)),
           lambda: ops.Linear(x, w, residual=torch.zeros((4, 3), device=dev)), lambda: ops.Linear(x, w, residual=x), lambda: ops.Linear(x, w.cpu()),
           lambda: ops.Linear(x, w, torch.zeros(3)), lambda: ops.Linear(x.int(), w.int()), lambda: ops.Linear(x.sum(), w)]
    for call in bad:
        with pytest.raises(ops.ChxqError):
            call()


# ---- LayerNormalization -----------------------------------------------------------------------------------------------------


def _norm64(x, scale, bias, eps):
    x = x.double()
    mean = x.mean(dim=-1, keepdim=True)
    inv = 1 / torch.sqrt(((x - mean) ** 2).mean(dim=-1, keepdim=True) + eps)
    y = (x - mean) * inv * scale.double()
    return (y if bias is None else y + bias.double()), mean, inv


def _check_norm(ops, dev, rows, d, dtype, affine, bias=True, shift=0.0, pitch=0, eps=1e-5):
    g = torch.Generator(device=dev).manual_seed(rows * 31 + d)
    x = (torch.randn((rows, d + pitch), device=dev, generator=g) * 1.5 + shift).to(dtype)[:, :d]
    scale, b = (torch.randn(d, device=dev, generator=g) + 1).to(affine), torch.randn(d, device=dev, generator=g).to(affine) if bias else None
    y, mean, inv = ops.LayerNormalization(x, scale, b, epsilon=eps, stats=True)
    assert y.dtype == dtype and y.is_contiguous() and mean.shape == inv.shape == (rows, 1) and mean.dtype == inv.dtype == torch.float32
    wy, wm, wi = _norm64(x, scale, b, eps)
    dm = (d + 2) * E32 * x.double().abs().mean(dim=1, keepdim=True)  # the mean's error
    _check(mean, wm, dm, "mean")
    # the variance: its own sum, and the mean's error twice (its square, since the deviations sum to zero, and the rounding of a deviation)
    dev_err = dm + E32 * (x.double().abs().amax(dim=1, keepdim=True) + wm.abs())
    var = 1 / wi ** 2
    rel = ((d + 6) * E32 * var + dm ** 2 + 2 * dev_err * var.sqrt()) / var
    _check(inv, wi, wi * (rel + EF), "inv_std_dev")
    xh = (x.double() - wm) * wi
    bound = scale.double().abs() * (dev_err * wi + xh.abs() * (rel + EF)) + EF * wy.abs() + (E32 * b.double().abs() if bias else 0)
    _check(y, wy, bound + _u(dtype) * 1.001 * wy.abs() + _tiny(dtype), "y %s" % ((rows, d, dtype),))
    assert torch.equal(ops.LayerNormalization(x, scale, b, epsilon=eps), y)
    return x, scale, mean, inv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 31), (1, 64), (7, 96), (64, 1000), (33, 1283), (2, 4096), (5, 8200), (3, 16384), (2, 40001), (3001, 256), (1200, 520)])
def test_layernorm_extents(ops, dev, dtype, rows, d):
    _check_norm(ops, dev, rows, d, dtype, dtype, bias=rows != 7)
    _check_norm(ops, dev, rows, d, dtype, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [1, 8])
def test_layernorm_shifted_rows_of_wider_buffers(ops, dev, dtype, pitch):
    """A mean far above the deviations: the variance is that of the deviations."""
    _check_norm(ops, dev, 50, 768, dtype, dtype, shift=100.0, pitch=pitch)


@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_axes_strides_and_constant_rows(ops, dev, dtype):
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((4, 6, 5, 8), device=dev, generator=g).to(dtype)
    s2, b2 = torch.randn((5, 8), device=dev, generator=g).to(dtype), torch.randn((5, 8), device=dev, generator=g).to(dtype)
    y, mean, inv = ops.LayerNormalization(x, s2, b2, axis=2, stats=True)
    assert mean.shape == inv.shape == (4, 6, 1, 1)
    flat = ops.LayerNormalization(x.view(24, 40), s2.view(40), b2.view(40))
    assert torch.equal(y.view(24, 40), flat) and torch.equal(ops.LayerNormalization(x, s2, b2, axis=-2), y)
    xp = x.permute(1, 0, 2, 3)
    assert torch.equal(ops.LayerNormalization(xp, s2, b2, axis=2), y.permute(1, 0, 2, 3))
    c = torch.full((3, 64), 2.5, dtype=dtype, device=dev)
    y, mean, inv = ops.LayerNormalization(c, s2.new_ones(64), s2.new_full((64,), 0.25), stats=True)
    assert torch.equal(y, torch.full_like(y, 0.25)) and torch.equal(mean, torch.full_like(mean, 2.5))
    _check(inv, torch.full((3, 1), 1e-5 ** -0.5, dtype=torch.float64, device=dev), 400 * EF)
    assert ops.LayerNormalization(c[:0], s2.new_ones(64)).shape == (0, 64)
    c[1, 5] = float("nan")
    y = ops.LayerNormalization(c, s2.new_ones(64), s2.new_full((64,), 0.25))
    assert torch.isnan(y[1]).all() and not torch.isnan(y[[0, 2]]).any()


@pytest.mark.parametrize("d", [64, 1000, 40000])
def test_layernorm_of_rows_whose_squares_overflow(ops, dev, d):
    """A variance that is infinite in 32 bits gives an inverse deviation of zero, not NaN, and leaves the other rows alone."""
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn((3, d), device=dev, generator=torch.Generator(device=dev).manual_seed(4)).to(dtype)
        x[1] = 1e25
        x[1, ::2] = -1e25
        s, b = torch.ones(d, device=dev), torch.full((d,), 0.5, device=dev)
        y, mean, inv = ops.LayerNormalization(x, s, b, stats=True)
        assert float(inv[1]) == 0 and float(mean[1].abs()) <= 1e25 and torch.equal(y[1], torch.full_like(y[1], 0.5))
        assert torch.equal(y[[0, 2]], ops.LayerNormalization(x[[0, 2]], s, b))


def _grad64(dy, x, scale, mean, inv):
    dy, xh = dy.double(), (x.double() - mean.double()) * inv.double()
    gd = dy * scale.double()
    dx = inv.double() * (gd - gd.mean(dim=-1, keepdim=True) - xh * (gd * xh).mean(dim=-1, keepdim=True))
    return dx, (dy * xh).sum(dim=0), dy.sum(dim=0)


def _check_grad(ops, dev, rows, d, dtype, affine, pitch=0):
    g = torch.Generator(device=dev).manual_seed(rows * 17 + d)
    x, dy = (torch.randn((rows, d + pitch), device=dev, generator=g).to(dtype)[:, :d] for _ in range(2))
    scale = (torch.randn(d, device=dev, generator=g) + 1).to(affine)
    mean = x.float().mean(dim=1, keepdim=True)
    inv = 1 / torch.sqrt((x.float() - mean).square().mean(dim=1, keepdim=True) + 1e-5)
    dx, ds, db = ops.LayerNormalizationGrad(dy, x, scale, mean, inv)
    assert dx.dtype == dtype and dx.is_contiguous() and ds.dtype == db.dtype == affine and ds.shape == db.shape == (d,)
    wx, ws, wb = _grad64(dy, x, scale, mean, inv)
    xh, gd = ((x.double() - mean.double()) * inv.double()).abs(), (dy.double() * scale.double()).abs()
    err = inv.double() * ((d + 8) * E32 * (gd.mean(dim=1, keepdim=True) + xh * (gd * xh).mean(dim=1, keepdim=True)) + 4 * E32 * gd) + EF * wx.abs()
    _check(dx, wx, err + _u(dtype) * 1.001 * wx.abs() + _tiny(dtype), "dx %s" % ((rows, d, dtype),))
    _check(ds, ws, (rows + 4) * E32 * (dy.double().abs() * xh).sum(dim=0) + _u(affine) * 1.001 * ws.abs() + _tiny(affine), "dscale")
    _check(db, wb, (rows + 4) * E32 * dy.double().abs().sum(dim=0) + _u(affine) * 1.001 * wb.abs() + _tiny(affine), "dbias")
    again = ops.LayerNormalizationGrad(dy, x, scale, mean, inv)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, ds, db)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 31), (64, 1000), (4099, 129), (301, 1283), (700, 4096), (5, 8200), (160, 16384), (3, 40001), (2001, 64)])
def test_layernorm_grad_extents(ops, dev, dtype, rows, d):
    _check_grad(ops, dev, rows, d, dtype, dtype)
    _check_grad(ops, dev, rows, d, dtype, torch.float32, pitch=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(20001, 520), (6001, 1030), (3001, 4999), (2405, 8192), (1501, 12001), (1203, 16384), (803, 28000), (171, 70001)])
def test_layernorm_grad_of_many_rows(ops, dev, dtype, rows, d):
    """More rows than a block holds at once, several times over: what holds the rows is filled again and again, and no wait runs out."""
    _check_grad(ops, dev, rows, d, dtype, dtype)
    ops.device_status()


def test_calls_from_two_threads(ops, dev):
    """Threads with a stream each call the same operators with other sizes, which need other amounts of shared memory, at the same time."""
    import threading

    g = torch.Generator(device=dev).manual_seed(9)
    cases = []
    for rows, d in ((300, 520), (200, 8192), (150, 4999), (90, 64)):
        x, dy = (torch.randn((rows, d), device=dev, generator=g) for _ in range(2))
        s = torch.randn(d, device=dev, generator=g)
        w = torch.randn((256, d), device=dev, generator=g)
        y, mean, inv = ops.LayerNormalization(x, s, stats=True)
        cases.append((x, dy, s, w, mean, inv, ops.LayerNormalizationGrad(dy, x, s, mean, inv), ops.Linear(y, w, activation="Tanh")))
    torch.cuda.synchronize()
    bad = []

    def work(order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in order * 25:
                    x, dy, s, w, mean, inv, want, z = cases[k]
                    got = ops.LayerNormalizationGrad(dy, x, s, mean, inv)
                    y = ops.LayerNormalization(x, s)
                    if not (all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(ops.Linear(y, w, activation="Tanh"), z)):
                        bad.append(k)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(o,)) for o in ([0, 1, 2, 3], [3, 2, 1, 0], [1, 0, 3, 2])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_layernorm_grad_against_differences(ops, dev):
    g = torch.Generator(device=dev).manual_seed(11)
    x, dy = torch.randn((6, 40), device=dev, generator=g), torch.randn((6, 40), device=dev, generator=g)
    scale, bias = torch.randn(40, device=dev, generator=g), torch.randn(40, device=dev, generator=g)
    y, mean, inv = ops.LayerNormalization(x, scale, bias, stats=True)
    dx, ds, db = ops.LayerNormalizationGrad(dy, x, scale, mean, inv)
    loss = lambda x, s, b: (_norm64(x, s, b, 1e-5)[0] * dy.double()).sum(dim=1)  # noqa: E731
    h = 1e-5  # differences in 64 bits: their error is about h^2 times a third derivative of a few tens, and 1e-16 / h
    for j in (0, 7, 39):
        e = torch.zeros(40, dtype=torch.float64, device=dev)
        e[j] = h
        d = (loss(x.double() + e, scale, bias) - loss(x.double() - e, scale, bias)) / (2 * h)
        assert (d - dx[:, j].double()).abs().max() < 1e-4
        d = ((loss(x, scale.double() + e, bias) - loss(x, scale.double() - e, bias)) / (2 * h)).sum()
        assert abs(float(d - ds[j])) < 1e-4
        d = ((loss(x, scale, bias.double() + e) - loss(x, scale, bias.double() - e)) / (2 * h)).sum()
        assert abs(float(d - db[j])) < 1e-4


@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_grad_of_broadcast_and_empty_inputs(ops, dev, dtype):
    """The gradient of a sum arrives expanded from one value; no rows give zero parameter gradients; the axis may cover several dimensions."""
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((3, 4, 6, 8), device=dev, generator=g).to(dtype)
    s = torch.randn((6, 8), device=dev, generator=g).to(dtype)
    _, mean, inv = ops.LayerNormalization(x, s, axis=2, stats=True)
    one = torch.ones((), dtype=dtype, device=dev).expand(x.shape)
    a = ops.LayerNormalizationGrad(one, x, s, mean, inv, axis=2)
    b = ops.LayerNormalizationGrad(one.contiguous().view(12, 48), x.view(12, 48), s.view(48), mean, inv)
    assert a[1].shape == (6, 8) and all(torch.equal(p.reshape(-1), q.reshape(-1)) for p, q in zip(a, b))
    e = ops.LayerNormalizationGrad(x[:0], x[:0], s, mean[:0], inv[:0], axis=2)
    assert e[0].shape == (0, 4, 6, 8) and not e[1].any() and not e[2].any()


def test_norm_refusals(ops, dev):
    x, s = torch.zeros((4, 8), dtype=torch.bfloat16, device=dev), torch.ones(8, device=dev)
    st = torch.zeros(4, device=dev)
    bad = [lambda: ops.LayerNormalization(x, s[:7]), lambda: ops.LayerNormalization(x, s.half()), lambda: ops.LayerNormalization(x, s, s.bfloat16()),
           lambda: ops.LayerNormalization(x, s, axis=2), lambda: ops.LayerNormalization(x, s, axis=-3), lambda: ops.LayerNormalization(x.int(), s),
           lambda: ops.LayerNormalization(x, s, epsilon=-1.0), lambda: ops.LayerNormalization(x, s, epsilon=float("nan")), lambda: ops.LayerNormalization(x[:, :0], s[:0]),
           lambda: ops.LayerNormalization(x, s, axis=0), lambda: ops.LayerNormalization(x, s.cpu()), lambda: ops.LayerNormalizationGrad(x[:2], x, s, st, st),
           lambda: ops.LayerNormalizationGrad(x.float(), x, s, st, st), lambda: ops.LayerNormalizationGrad(x, x, s, st[:3], st),
           lambda: ops.LayerNormalizationGrad(x, x, s, st, st.double()), lambda: ops.LayerNormalizationGrad(x, x, s, st.cpu(), st)]
    for call in bad:
        with pytest.raises(ops.ChxqError):
            call()


# ---- TokenLogProbs ----------------------------------------------------------------------------------------------------------


def _logprobs64(x, tok):
    x = x.double()
    logp = torch.log_softmax(x, dim=-1)
    p = torch.exp(logp)
    ent = torch.special.entr(p).sum(dim=-1)
    lse = torch.logsumexp(x, dim=-1)
    return logp, logp.gather(1, tok.long()[:, None])[:, 0], ent, lse


def _check_logprobs(ops, dev, x, tok, k):
    """The sum of the exponentials is off by (V 2^-23 + EF) relative, so its log by as much absolutely, next to the roundings of lse itself and
    of the differences; the entropy's two parts the same, times the size of the largest exponent that has a share (log V + a few)."""
    rows, v = x.shape
    lp, ent, lse, top_lp, top = ops.TokenLogProbs(x, tok, k)
    logp, wlp, went, wlse = _logprobs64(x, tok)
    rel = v * E32 + EF
    scale = wlse.abs() + x.double().masked_fill(torch.isinf(x), 0).abs().amax(dim=1)
    _check(lse, wlse, rel + 4 * E32 * scale, "log_sum_exp")
    spread = (x.double().amax(dim=1) - x.double().gather(1, tok.long()[:, None])[:, 0]).abs()  # lp = (x - max) - log sum
    _check(lp, wlp, rel + 8 * E32 * (spread + math.log(v) + 1), "logprob")
    _check(ent, went, (rel + 8 * E32 * scale) * (math.log(v) + 20), "entropy")
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    assert top.dtype == torch.int64 and torch.equal(top, order)
    _check(top_lp, logp.gather(1, order), rel + 8 * E32 * (2 * logp.gather(1, order).abs() + math.log(v) + 1), "top log probabilities")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (2, 7, 7), (5, 10, 3), (256, 1000, 5), (3, 33, 32), (64, 777, 1), (1, 32000, 20), (4, 50001, 32), (1, 131072, 20), (300, 4097, 0),
                                      (2, 262144, 5), (1500, 129, 8)])
def test_token_logprobs_extents(ops, dev, dtype, rows, v, k):
    g = torch.Generator(device=dev).manual_seed(rows + v)
    x = (torch.randn((rows, v), device=dev, generator=g) * 3).to(dtype)
    _check_logprobs(ops, dev, x, torch.randint(0, v, (rows,), device=dev, generator=g), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "few values", "lowest", "forbidden", "spike"])
def test_token_logprobs_orders_and_masks(ops, dev, dtype, kind):
    rows, v, k = 6, 9001, 20
    g = torch.Generator(device=dev).manual_seed(4)
    x = (torch.randn((rows, v), device=dev, generator=g) * 3).to(dtype)
    tok = torch.randint(0, v, (rows,), device=dev, generator=g)
    if kind in ("ascending", "descending"):
        x = torch.sort(x, dim=1, descending=kind == "descending")[0]
    elif kind == "equal":
        x = torch.full_like(x, -7.25)
    elif kind == "few values":
        x = torch.randint(0, 3, (rows, v), device=dev, generator=g).to(dtype)
    elif kind == "lowest":
        x[torch.rand((rows, v), device=dev, generator=g) < 0.9] = torch.finfo(dtype).min
        x[0] = torch.finfo(dtype).min
        x[1:, 17] = 1.0
        tok[1:] = 17
    elif kind == "forbidden":
        x[torch.rand((rows, v), device=dev, generator=g) < 0.999] = float("-inf")
        x[:, 8000] = 2.0
        x[1] = float("-inf")
        x[1, 5] = -3.0
        tok[:] = 8000
        tok[1] = 5
    else:
        x[:, 4321] = 30000.0
        tok[:3] = 4321
    _check_logprobs(ops, dev, x, tok, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_special_rows_and_tokens(ops, dev, dtype):
    v = 5000
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn((6, v), device=dev, generator=g).to(dtype)
    x[1] = float("-inf")
    x[2, 77] = float("nan")
    x[3, 4999] = float("inf")
    tok = torch.tensor([5, 5, 6, 4999, -1, v], device=dev)
    lp, ent, lse, top_lp, top = ops.TokenLogProbs(x, tok, 4)
    assert float(lp[1]) == float(lse[1]) == -math.inf and float(ent[1]) == 0 and top[1].tolist() == [0, 1, 2, 3] and (top_lp[1] == -math.inf).all()
    for r in (2, 3):
        assert all(torch.isnan(t[r]).all() for t in (lp, ent, lse, top_lp))
    assert int(top[2, 0]) == 77 and int(top[3, 0]) == 4999
    assert torch.isnan(lp[4]) and torch.isnan(lp[5]) and not torch.isnan(ent[4:]).any()
    lp2, ent2, *_ = ops.TokenLogProbs(x, tok, 0, ignore_index=-1)
    assert float(lp2[4]) == 0 and torch.isnan(lp2[5]) and torch.equal(ent2[4:], ent[4:]) and torch.equal(lp2[:1], lp[:1])
    lp3 = ops.TokenLogProbs(x, tok.int(), 2, ignore_index=5)[0]
    assert float(lp3[0]) == 0 and float(lp3[1]) == 0 and torch.isnan(lp3[2])
    d = ops.TokenLogProbsGrad(torch.ones(6, device=dev), None, x, tok, lse, ent, ignore_index=-1).float()
    assert not d[1, 6:].any() and torch.isnan(d[2]).all() and not d[4].any() and torch.isnan(d[5]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 3])
def test_token_logprobs_rows_of_wider_buffers(ops, dev, dtype, shift):
    g = torch.Generator(device=dev).manual_seed(shift)
    buf = (torch.randn((20, 3, 1003), device=dev, generator=g) * 2).to(dtype)
    x, tok = buf[:, 1, shift:1001], torch.randint(0, 1001 - shift, (20,), device=dev, generator=g)
    _check_logprobs(ops, dev, x, tok, 6)
    a = ops.TokenLogProbs(buf[:, :, shift:1001], tok[:, None].expand(20, 3), 6)
    assert a[0].shape == (20, 3) and a[4].shape == (20, 3, 6)
    b = ops.TokenLogProbs(x, tok, 6)
    assert all(torch.equal(p[:, 1], q) for p, q in zip(a, b))
    assert ops.TokenLogProbs(x[:0], tok[:0], 2)[3].shape == (0, 2)


def _check_logprobs_grad(ops, dev, x, tok, seed=0):
    rows, v = x.shape
    g = torch.Generator(device=dev).manual_seed(seed)
    dlp, dent = torch.randn(rows, device=dev, generator=g), torch.randn(rows, device=dev, generator=g)
    lp, ent, lse, _, _ = ops.TokenLogProbs(x, tok)
    d = ops.TokenLogProbsGrad(dlp, dent, x, tok, lse, ent)
    assert d.shape == x.shape and d.dtype == x.dtype and d.is_contiguous()
    logp = x.double() - lse.double()[:, None]
    p = torch.exp(logp)
    inner = torch.nan_to_num(p * logp, nan=0.0) + p * ent.double()[:, None]
    hot = torch.zeros_like(p).scatter_(1, tok.long()[:, None], 1.0)
    want = dlp.double()[:, None] * (hot - p) - dent.double()[:, None] * inner
    # log p is off by a rounding of itself, which is relative in p and absolute in the second term
    dl = 2 * E32 * logp.masked_fill(torch.isinf(logp), 0).abs() + EF
    bound = dl * p * (dlp.double().abs()[:, None] + dent.double().abs()[:, None] * (logp.masked_fill(torch.isinf(logp), 0).abs() + ent.double()[:, None] + 2))
    _check(d, want, bound + 4 * E32 * want.abs() + _u(x.dtype) * 1.001 * want.abs() + _tiny(x.dtype), "dlogits")
    a, b = ops.TokenLogProbsGrad(dlp, None, x, tok, lse), ops.TokenLogProbsGrad(None, dent, x, tok, lse, ent)
    _check(a, dlp.double()[:, None] * (hot - p), bound + _u(x.dtype) * 1.01 * (dlp.double()[:, None] * (hot - p)).abs() + _tiny(x.dtype), "dlogprob alone")
    _check(b, -dent.double()[:, None] * inner, bound + _u(x.dtype) * 1.01 * (dent.double()[:, None] * inner).abs() + _tiny(x.dtype), "dentropy alone")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 7), (256, 1000), (5, 1001), (2, 50001), (1, 131072), (700, 129), (2003, 303), (77, 509), (77, 510), (9, 1017), (9, 1018), (41, 13)])
def test_token_logprobs_grad_extents(ops, dev, dtype, rows, v):
    g = torch.Generator(device=dev).manual_seed(rows * 3 + v)
    x = (torch.randn((rows, v), device=dev, generator=g) * 3).to(dtype)
    tok = torch.randint(0, v, (rows,), device=dev, generator=g)
    _check_logprobs_grad(ops, dev, x, tok)
    if v > 8:
        x[:, ::3] = float("-inf")
        _check_logprobs_grad(ops, dev, x, torch.full_like(tok, 1))
        wide = (torch.randn((rows, v + 5), device=dev, generator=g) * 3).to(dtype)
        _check_logprobs_grad(ops, dev, wide[:, 3:v + 3], tok.int())


@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_grad_of_rows_far_from_zero(ops, dev, dtype):
    """log_sum_exp of such a row has lost the digits of the probabilities: rows of nothing but the type's lowest value are uniform all the same."""
    v = 1000
    x = torch.full((3, v), torch.finfo(dtype).min, dtype=dtype, device=dev)
    x[1] = torch.finfo(dtype).max
    x[2, 7:] = float("-inf")
    tok = torch.tensor([3, 4, 5], device=dev)
    _, ent, lse, _, _ = ops.TokenLogProbs(x, tok)
    d = ops.TokenLogProbsGrad(torch.ones(3, device=dev), torch.ones(3, device=dev), x, tok, lse, ent)
    want = torch.zeros((3, v), dtype=torch.float64, device=dev)
    want[:2], want[2, :7] = -1.0 / v, -1.0 / 7
    want[torch.arange(3), tok] += 1  # a uniform row's entropy is stationary
    _check(d, want, v * E32 * want.abs() + 100 * EF / v + _u(dtype) * 1.01 * want.abs() + _tiny(dtype))


def test_token_logprobs_grad_against_differences(ops, dev):
    g = torch.Generator(device=dev).manual_seed(1)
    x, tok = torch.randn((4, 30), device=dev, generator=g), torch.randint(0, 30, (4,), device=dev, generator=g)
    dlp, dent = torch.randn(4, device=dev, generator=g), torch.randn(4, device=dev, generator=g)
    _, ent, lse, _, _ = ops.TokenLogProbs(x, tok)
    d = ops.TokenLogProbsGrad(dlp, dent, x, tok, lse, ent)

    def loss(z):
        _, lp, en, _ = _logprobs64(z, tok)
        return dlp.double() * lp + dent.double() * en
    for j in range(30):
        e = torch.zeros(30, dtype=torch.float64, device=dev)
        e[j] = 1e-5
        assert ((loss(x.double() + e) - loss(x.double() - e)) / 2e-5 - d[:, j].double()).abs().max() < 1e-5


def test_logprob_refusals(ops, dev):
    x, t, f = torch.zeros((4, 8), device=dev), torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(4, device=dev)
    bad = [lambda: ops.TokenLogProbs(x, t, 9), lambda: ops.TokenLogProbs(torch.zeros((4, 64), device=dev), t, 33), lambda: ops.TokenLogProbs(x, t, -1),
           lambda: ops.TokenLogProbs(x, t[:3]), lambda: ops.TokenLogProbs(x, f), lambda: ops.TokenLogProbs(x.int(), t), lambda: ops.TokenLogProbs(x[:, :0], t),
           lambda: ops.TokenLogProbs(x, t.cpu()), lambda: ops.TokenLogProbs(x.sum(), t), lambda: ops.TokenLogProbsGrad(f, f, x, t, f),
           lambda: ops.TokenLogProbsGrad(f[:2], None, x, t, f), lambda: ops.TokenLogProbsGrad(f, None, x, t, f.double()), lambda: ops.TokenLogProbsGrad(f.cpu(), None, x, t, f)]
    for call in bad:
        with pytest.raises(ops.ChxqError):
            call()


# ---- together ---------------------------------------------------------------------------------------------------------------


def _block(ops, h, p, tok):
    """Norm, product with activation, product with residual, norm, product to the logits, log probabilities."""
    n1, m1, i1 = ops.LayerNormalization(h, p["s1"], p["b1"], stats=True)
    u = ops.Linear(n1, p["w1"], p["c1"], activation="GeluTanh")
    h2 = ops.Linear(u, p["w2"], p["c2"], residual=h)
    n2, m2, i2 = ops.LayerNormalization(h2, p["s2"], p["b2"], stats=True)
    logits = ops.Linear(n2, p["wv"], residual=p["rv"])
    return h2, m2, i2, logits, ops.TokenLogProbs(logits, tok, 5)


def _params(dev, dtype, d=256, f=512, v=1000, rows=48, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, device=dev, generator=g)  # noqa: E731
    p = {"s1": r(d) * 0.1 + 1, "b1": r(d) * 0.1, "w1": r(f, d) / 16, "c1": r(f) * 0.1, "w2": r(d, f) / 22, "c2": r(d) * 0.1, "s2": r(d) * 0.1 + 1, "b2": r(d) * 0.1,
         "wv": r(v, d) / 8, "rv": r(rows, v) * 0.1}
    return {k: t.to(dtype) for k, t in p.items()}, r(rows, d).to(dtype), torch.randint(0, v, (rows,), device=dev, generator=g)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_block_with_the_gradients_of_its_end(ops, dev, dtype):
    """Forward through all the operators, then back from the log probabilities through the logits' product (on the transposed weights) to the second
    norm, against the same block in 64 bits by automatic differentiation.  16-bit types round at six places on the way; each is a relative
    half step, and the last is followed by the sums of the next product, so a few steps of the norm of the result are allowed."""
    p, h, tok = _params(dev, dtype)
    h2, m2, i2, logits, (lp, ent, lse, top_lp, top) = _block(ops, h, p, tok)
    rows = h.shape[0]
    dlogits = ops.TokenLogProbsGrad(torch.full((rows,), -1.0 / rows, device=dev), None, logits, tok, lse)
    dn2 = ops.Linear(dlogits, p["wv"].t())
    dh2, ds, db = ops.LayerNormalizationGrad(dn2, h2, p["s2"], m2, i2)
    q = {k: t.double() for k, t in p.items()}
    x2 = h2.double().requires_grad_()
    s2, b2 = q["s2"].clone().requires_grad_(), q["b2"].clone().requires_grad_()
    want_logits = _norm64(x2, s2, b2, 1e-5)[0] @ q["wv"].t() + q["rv"]
    n1 = _norm64(h, q["s1"], q["b1"], 1e-5)[0]
    want_h2 = _act64(n1 @ q["w1"].t() + q["c1"], "GeluTanh") @ q["w2"].t() + q["c2"] + h.double()
    loss = -torch.log_softmax(want_logits, dim=1).gather(1, tok[:, None]).mean()
    loss.backward()
    near = lambda a, b, steps: float((a.double() - b).norm() / b.norm()) <= steps * _u(dtype) + 2e-6  # noqa: E731
    assert near(h2, want_h2, 3) and near(logits, want_logits.detach(), 3) and near(-lp.mean(), loss.detach(), 3)
    assert near(dh2, x2.grad, 6) and near(ds, s2.grad, 6) and near(db, b2.grad, 6)


def test_a_block_captured_and_replayed_beside_another_stream(ops, dev):
    """The same bits from a captured graph with new inputs, while another stream runs the operators on other data."""
    p, h, tok = _params(dev, torch.bfloat16)
    _, h_new, tok_new = _params(dev, torch.bfloat16, seed=1)
    flat = lambda out: [out[0], out[1], out[2], out[3], *out[4]]  # noqa: E731
    want, want_new = [t.clone() for t in flat(_block(ops, h, p, tok))], [t.clone() for t in flat(_block(ops, h_new, p, tok_new))]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(ops, h, p, tok)
    torch.cuda.current_stream().wait_stream(side)
    hs, ts = h.clone(), tok.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = flat(_block(ops, hs, p, ts))
    for src, t, w in ((h_new, tok_new, want_new), (h, tok, want)):
        hs.copy_(src)
        ts.copy_(t)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = flat(_block(ops, h_new, p, tok_new))
        graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, w)) and all(torch.equal(a, b) for a, b in zip(other, want_new))
    ops.device_status()


def test_offsets_past_32_bits(ops, dev):
    """More than 2^31 values in the operands and results: the last rows are those of a small call."""
    def ends(full, part, rows):
        return torch.equal(full[-rows:], part)

    g = torch.Generator(device=dev).manual_seed(3)
    x, w, r = torch.randn((70001, 16), device=dev, generator=g).bfloat16(), torch.randn((32768, 16), device=dev, generator=g).bfloat16(), None
    y = ops.Linear(x, w, activation="Relu")  # 2.3e9 outputs
    want, bound = _linear64(x[-200:], w, None, "Relu", r, False)
    _check(y[-200:], want, bound)
    del y
    x = torch.empty((131100, 16411), dtype=torch.bfloat16, device=dev)  # 2.15e9
    part = torch.randn((300, 16411), device=dev, generator=g).bfloat16()
    x[:], x[-300:] = 1.0, part
    s = torch.randn(16411, device=dev, generator=g)
    y, mean, inv = ops.LayerNormalization(x, s, stats=True)
    py, pm, pi = ops.LayerNormalization(part, s, stats=True)
    assert torch.equal(mean[-300:], pm) and torch.equal(inv[-300:], pi) and torch.equal(y[-300:], py)
    dx = ops.LayerNormalizationGrad(x, x, s, mean, inv)[0]
    assert ends(dx[-290:-10], ops.LayerNormalizationGrad(part, part, s, pm, pi)[0][10:-10], 280)
    del dx, y
    tok = torch.randint(0, 16411, (131100,), device=dev, generator=g)
    lp, ent, lse, tl, tt = ops.TokenLogProbs(x, tok, 3)
    a = ops.TokenLogProbs(part, tok[-300:], 3)
    ref = torch.log_softmax(part.double(), dim=1).gather(1, tok[-300:, None])[:, 0]
    sums = (16411 + 16) * E32  # of a row, and its logarithm
    assert ((lp[-300:].double() - ref).abs() <= sums + 4 * E32 * ref.abs()).all() and torch.equal(tt[-300:], a[4])
    assert ((lse[-300:] - a[2]).abs() <= 2 * sums + 2 * E32 * a[2].abs()).all()
    one = torch.ones(131100, device=dev)
    d = ops.TokenLogProbsGrad(one, None, x, tok, lse)
    assert ends(d, ops.TokenLogProbsGrad(one[-300:], None, part, tok[-300:], lse[-300:]), 300)
