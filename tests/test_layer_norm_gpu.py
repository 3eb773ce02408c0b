"""GPU parity: layer norm of rows, forward and backward, against its definition in float64.

Error bounds, per entry.  u = half a step of the type, e = 2^-24, C = width, n = rows.
forward   mean: C e (mean |x|) summed in fp32 in an order not ours; a difference d = x - mean is off by dm = (C + 2) e mean|x| + e |d|;
          the variance by that and (C + 3) e of itself, so rstd by r = (C + 6) e + dm rstd, relative;
          y by |w| rstd (dm + |d| r) + 4 e (|w u| + |b|), and u |y| for its rounding.
backward  v = d rstd is off by dv = rstd dm + |v| r; g by e |g|; the row's means by (C + 4) e mean|g| and mean|g| max dv + (C + 4) e mean|g v|;
          dx = rstd (g - m1 - v m2) by the sum of those, r of itself, 6 e of its terms, u |dx|.
          dw: sum over rows of |dy| dv + (n + 4) e |dy v|, and u; db: (n + 2) e sum |dy|, and u.
"""
import pytest
import torch

import acnative

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
KINDS = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _u(kind):
    return torch.finfo(kind).eps / 2


def _make(rows, C, kind, wkind, seed=0, shift=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * 1.3 + shift * torch.randn(C, generator=g)).to(KINDS[kind])
    dy = torch.randn(rows, C, generator=g).to(KINDS[kind])
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(KINDS[wkind])
    b = (0.5 * torch.randn(C, generator=g)).to(KINDS[wkind])
    return x, dy, w, b


def _reference(x, dy, w, b, eps):
    C = x.shape[1]
    x, dy = x.double(), dy.double()
    wd = torch.ones(C, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    v, g = d * rstd, dy * wd
    m1, m2 = g.mean(1, keepdim=True), (g * v).mean(1, keepdim=True)
    r = {"mean": mean[:, 0], "rstd": rstd[:, 0], "y": v * wd + bd, "dx": rstd * (g - m1 - v * m2), "dw": (dy * v).sum(0), "db": dy.sum(0)}
    dm = (C + 2) * E * x.abs().mean(1, keepdim=True) + E * d.abs()
    dm0 = dm.amax(1, keepdim=True)
    rel = (C + 6) * E + dm0 * rstd
    dv = rstd * dm + v.abs() * rel
    n = x.shape[0]
    t = {"mean": ((C + 2) * E * x.abs().mean(1)), "rstd": rstd[:, 0] * rel[:, 0], "y": wd.abs() * dv + 4 * E * ((wd * v).abs() + bd.abs()),
         "dw": (dy.abs() * dv).sum(0) + (n + 4) * E * (dy * v).abs().sum(0), "db": (n + 2) * E * dy.abs().sum(0)}
    ga = g.abs().mean(1, keepdim=True)
    e1 = (C + 4) * E * ga
    e2 = (g.abs() * dv).mean(1, keepdim=True) + (C + 4) * E * (g * v).abs().mean(1, keepdim=True)
    t["dx"] = rstd * (e1 + v.abs() * e2 + dv * m2.abs() + 6 * E * (g.abs() + m1.abs() + (v * m2).abs())) + r["dx"].abs() * rel
    return r, t


def _check(name, got, ref, tol, kind):
    got = got.cpu().double()
    bound = tol + _u(kind) * ref.abs() + (2.0 ** -25 if kind == torch.float16 else 1e-37)
    assert got.shape == ref.shape and torch.isfinite(got).all(), name
    assert ((got - ref).abs() <= bound).all(), "%s: error %.3g of its bound" % (name, ((got - ref).abs() / bound).max())


def _all(dev, rows, C, kind, wkind, w=True, b=True, eps=1e-6, seed=0, shift=1.0):
    x, dy, W, B = _make(rows, C, kind, wkind, seed, shift)
    W, B = W if w else None, B if b else None
    r, t = _reference(x, dy, W, B, eps)
    to = lambda v: None if v is None else v.to(dev)  # noqa: E731
    y, mean, rstd = acnative.layer_norm(x.to(dev), to(W), to(B), eps=eps, want_stats=True)
    dx, dw, db = acnative.layer_norm_backward(dy.to(dev), x.to(dev), to(W), mean, rstd)
    what = "%d x %d %s/%s " % (rows, C, kind, wkind)
    _check(what + "mean", mean, r["mean"], t["mean"], torch.float32)
    _check(what + "rstd", rstd, r["rstd"], t["rstd"], torch.float32)
    _check(what + "y", y, r["y"], t["y"], x.dtype)
    _check(what + "dx", dx, r["dx"], t["dx"], x.dtype)
    wtype = W.dtype if w else torch.float32
    assert dw.dtype == db.dtype == wtype
    _check(what + "dw", dw, r["dw"], t["dw"], wtype)
    _check(what + "db", db, r["db"], t["db"], wtype)


@pytest.mark.parametrize("kind,wkind", [("fp32", "fp32"), ("fp16", "fp16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp32")])
@pytest.mark.parametrize("C", [1, 2, 7, 64, 65, 192, 512, 768, 1000, 1024, 1032, 2050, 4096, 4100, 5120, 8192, 12289, 16384, 16392, 20001])
def test_widths(dev, kind, wkind, C):
    _all(dev, 37, C, kind, wkind, seed=C)
    _all(dev, 1, C, kind, wkind, seed=C + 1)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [2, 3, 4, 5, 255, 1023, 1025, 5000])
def test_rows(dev, kind, rows):
    _all(dev, rows, 192, kind, kind, seed=rows)
    _all(dev, rows, 1288, kind, "fp32", seed=rows)


def test_without_weights_large_means_and_eps(dev):
    _all(dev, 9, 320, "bf16", "bf16", w=False, b=False)
    _all(dev, 9, 320, "fp32", "fp32", b=False)
    _all(dev, 9, 320, "fp16", "fp32", w=False)
    _all(dev, 50, 768, "fp32", "fp32", shift=100.0)                    # the means dwarf the differences
    _all(dev, 50, 768, "fp32", "fp32", eps=0.5)
    x = torch.full((3, 256), 2.5, device=dev)                          # no variance: y is the bias
    b = torch.arange(256.0, device=dev)
    assert torch.equal(acnative.layer_norm(x, torch.ones(256, device=dev), b), b.expand(3, 256))


def test_strides_shapes_in_place_and_parts(dev):
    x, dy, w, b = _make(24, 96, "bf16", "bf16", 3)
    r, t = _reference(x, dy, w, b, 1e-6)
    wide = torch.full((24, 200), 9.0, dtype=torch.bfloat16, device=dev)
    for at in (8, 5):                                                  # 16-byte rows, then odd ones
        view = wide[:, at:at + 96]
        view.copy_(x.to(dev))
        y, mean, rstd = acnative.layer_norm(view, w.to(dev), b.to(dev), want_stats=True)
        _check("y", y, r["y"], t["y"], x.dtype)
        dx, dw, db = acnative.layer_norm_backward(dy.to(dev), view, w.to(dev), mean, rstd)
        for name, v in (("dx", dx), ("dw", dw), ("db", db)):
            _check(name, v, r[name], t[name], x.dtype)
        only = acnative.layer_norm_backward(dy.to(dev), view, w.to(dev), mean, rstd, want=(False, True, False))
        assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
        only = acnative.layer_norm_backward(dy.to(dev), view, w.to(dev), mean, rstd, want=(True, False, False))
        assert torch.equal(only[0], dx) and only[1] is None
        out = acnative.layer_norm(view, w.to(dev), b.to(dev), out=view)
        assert out is view and torch.equal(view, y)
        assert (wide[:, :at] == 9.0).all() and (wide[:, at + 96:] == 9.0).all()
        wide.fill_(9.0)
    three = x.to(dev).reshape(2, 12, 96)
    y3, m3, s3 = acnative.layer_norm(three, w.to(dev), b.to(dev), want_stats=True)
    assert y3.shape == three.shape and m3.shape == (2, 12)
    _check("y", y3.reshape(24, 96), r["y"], t["y"], x.dtype)
    turned = x.to(dev).reshape(2, 12, 96).transpose(0, 1)              # axes that do not fold: copied
    _check("y", acnative.layer_norm(turned, w.to(dev), b.to(dev)).transpose(0, 1).reshape(24, 96), r["y"], t["y"], x.dtype)
    one = x.to(dev)[:1].expand(24, 96)
    assert torch.equal(acnative.layer_norm(one, w.to(dev), b.to(dev))[7], acnative.layer_norm(x.to(dev)[:1], w.to(dev), b.to(dev))[0])


def test_no_rows(dev):
    x = torch.zeros(0, 64, device=dev)
    w = torch.ones(64, device=dev)
    y, mean, rstd = acnative.layer_norm(x, w, w, want_stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = acnative.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_infinities_and_nan_stay_in_their_row(dev):
    x, dy, w, b = _make(10, 256, "fp32", "fp32", 5)
    want, mean, rstd = acnative.layer_norm(x.to(dev), w.to(dev), b.to(dev), want_stats=True)
    dirty = x.clone()
    dirty[3, 7], dirty[6, 0] = float("inf"), float("nan")
    got, m2, r2 = acnative.layer_norm(dirty.to(dev), w.to(dev), b.to(dev), want_stats=True)
    keep = [i for i in range(10) if i not in (3, 6)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[6]).all() and torch.isnan(got[3]).all()
    a = acnative.layer_norm_backward(dy.to(dev), x.to(dev), w.to(dev), mean, rstd)[0]
    c = acnative.layer_norm_backward(dy.to(dev), dirty.to(dev), w.to(dev), m2, r2)[0]
    assert torch.equal(a[keep], c[keep]) and torch.isnan(c[3]).all()


def test_gradients_against_differences(dev):
    """Central differences of the fp32 forward pass along random directions."""
    x, dy, w, b = (t.to(dev) for t in _make(6, 200, "fp32", "fp32", 8))
    y, mean, rstd = acnative.layer_norm(x, w, b, want_stats=True)
    grads = acnative.layer_norm_backward(dy, x, w, mean, rstd)
    g = torch.Generator().manual_seed(1)
    h = 1e-2
    for i, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g).to(dev)
        args = lambda s: [u + s * h * d if u is t else u for u in (x, w, b)]  # noqa: E731
        up, down = acnative.layer_norm(*args(1)).double(), acnative.layer_norm(*args(-1)).double()
        slope = ((up - down) * dy.double()).sum() / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        # the difference's own error: third derivatives h^2 / 6 (of a map of order one, 1200 terms) and rounding 2^-23 / h each
        assert abs(slope - want) <= 1200 ** 0.5 * (10 * h * h + 4 * 2.0 ** -23 / h * 4)


def test_same_bits_every_time_and_in_a_graph(dev):
    x, dy, w, b = (t.to(dev) for t in _make(3001, 768, "bf16", "fp32", 9))

    def step():
        y, mean, rstd = acnative.layer_norm(x, w, b, want_stats=True)
        return (y,) + acnative.layer_norm_backward(dy, x, w, mean, rstd)
    first = step()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, step()))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    for turn in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
        x.mul_(1.5)
        torch.cuda.synchronize()


def test_more_rows_than_one_launch_takes(dev):
    n = (1 << 25) + 5                                               # 8 threads to a row, 2^28 to a launch
    gen = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((n, 3), generator=gen, device=dev).bfloat16()
    w = torch.randn(3, generator=gen, device=dev)
    y, mean, rstd = acnative.layer_norm(x, w, w, want_stats=True)
    for a, b in ((0, 9), ((1 << 25) - 7, n)):
        part = acnative.layer_norm(x[a:b], w, w, want_stats=True)
        for whole, p in zip((y, mean, rstd), part):
            assert torch.equal(whole[a:b], p)


def test_more_wide_rows_than_one_launch_takes(dev):
    n, C = (1 << 18) + 3, 16392                                     # 1024 threads to a row; one row taken n times
    gen = torch.Generator(device=dev).manual_seed(6)
    x, dy = (torch.randn((1, C), generator=gen, device=dev).bfloat16() for _ in range(2))
    w = torch.randn(C, generator=gen, device=dev)
    _, mean, rstd = acnative.layer_norm(x, w, w, want_stats=True)
    one = acnative.layer_norm_backward(dy, x, w, mean, rstd, want=(True, False, False))[0]
    dx = acnative.layer_norm_backward(dy.expand(n, C), x.expand(n, C), w, mean.repeat(n), rstd.repeat(n), want=(True, False, False))[0]
    for i in (0, (1 << 18) - 1, 1 << 18, n - 1):
        assert torch.equal(dx[i], one[0]), i
