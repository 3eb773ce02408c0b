"""GPU parity: forms and plans of the packed-sequence operators that test_packed_gpu.py does not reach (its bounds hold here too)."""
import math

import pytest
import torch

import acnative
from oracle import packed as opacked
from test_packed_gpu import E, KINDS, _check_attention, _randn, _run, _starts, _u

pytestmark = pytest.mark.gpu


def _check_rotary(got, x, pos, freq, layout, offset, amplitude, kind, inverse=False):
    ref, size = opacked.rotary(x, pos, freq, layout, offset, amplitude, inverse)
    tol = _u(kind) * ref.abs() + (2.0 ** -22 + 4 * E) * size + (2.0 ** -25 if kind == "fp16" else 0.0)
    assert ((got.cpu().double() - ref).abs() <= tol).all()


# ----------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D,part,offset", [(48, 48, 0), (80, 24, 8), (37, 20, 6), (3, 2, 0), (300, 10, 286)])
def test_rotary_interleaved_on_odd_strides(dev, kind, D, part, offset):
    """Heads that start at odd entries, odd head sizes: a slice of [tokens, heads, dim + 3], turned beside itself and in place."""
    T, H, G = 19, 4, 2
    base = _randn((T + 1, H + G + 1, D + 3), D, kind)
    x, xk = base[1:, 1:H + 1, 3:], base[1:, H + 1:, 3:]
    pos = torch.randint(0, 100000, (T,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    freq = acnative.rotary_frequencies(part)
    d = base.to(dev)
    q, k = d[1:, 1:H + 1, 3:], d[1:, H + 1:, 3:]
    args = (pos.to(dev), freq.to(dev))
    for a, b in zip(acnative.rotary(q, k, *args, layout="interleaved", offset=offset, amplitude=0.75), (x, xk)):
        _check_rotary(a, b, pos, freq, "interleaved", offset, 0.75, kind)
    acnative.rotary(q, k, *args, layout="interleaved", offset=offset, amplitude=0.75, out_q=q, out_k=k)
    _check_rotary(q, x, pos, freq, "interleaved", offset, 0.75, kind)
    _check_rotary(k, xk, pos, freq, "interleaved", offset, 0.75, kind)
    rest = torch.ones(base.shape, dtype=torch.bool)
    rest[1:, 1:, 3 + offset:3 + offset + part] = False
    assert torch.equal(d.cpu()[rest], base[rest])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_of_axes_of_one(dev, layout):
    """A tensor of one token or one head may carry any stride for that axis."""
    base = _randn((3, 5, 64), 1, "bf16")
    d = base.to(dev)
    freq = acnative.rotary_frequencies(64)
    pos = torch.tensor([123, 7, 99], dtype=torch.int32)
    one = d.as_strided((1, 5, 64), (321, 64, 1))
    out = torch.zeros(400, dtype=torch.bfloat16, device=dev).as_strided((1, 5, 64), (333, 64, 1))
    acnative.rotary(one, None, pos[:1].to(dev), freq.to(dev), layout=layout, out_q=out)
    _check_rotary(out, base[:1], pos[:1], freq, layout, 0, 1.0, "bf16")
    head = d.as_strided((3, 1, 64), (320, 7, 1))
    got = acnative.rotary(head, head, pos.to(dev), freq.to(dev), layout=layout)
    for y in got:
        _check_rotary(y, base[:, :1], pos, freq, layout, 0, 1.0, "bf16")


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_turned_back(dev, kind, layout):
    """inverse=True is the transpose of the map, amplitude included: against the oracle, and <y, R x> = <R^T y, x>."""
    T, H, G, D, part, offset = 45, 4, 2, 80, 48, 16
    x, y = _randn((T, H, D), 1, kind), _randn((T, G, D), 2, kind)
    pos = torch.randint(-5, 4_000_000, (2, T), generator=torch.Generator().manual_seed(3), dtype=torch.int64)
    freq = acnative.rotary_frequencies(part, 10000.0, axes=2, factor=4.0, original=2048)
    args = {"layout": layout, "offset": offset, "amplitude": 1.25}
    got = acnative.rotary(x.to(dev), y.to(dev), pos.to(dev), freq.to(dev), inverse=True, **args)
    for a, b in zip(got, (x, y)):
        _check_rotary(a, b, pos, freq, layout, offset, 1.25, kind, inverse=True)
    if kind == "fp32":
        y = _randn((T, H, D), 4, kind)
        turned = acnative.rotary(x.to(dev), None, pos.to(dev), freq.to(dev), **args).cpu().double()
        back = acnative.rotary(y.to(dev), None, pos.to(dev), freq.to(dev), inverse=True, **args).cpu().double()
        # each entry of either is off by the bound of _check_rotary: below 2^-21 of the two magnitudes behind it, times 1.25 for the amplitude
        slack = 2 * 2.0 ** -21 * 1.25 * 2 * (x.double().abs().amax(-1) * y.double().abs().amax(-1)).sum() * D
        assert abs((y.double() * turned).sum() - (back * x.double()).sum()) <= slack


# ------------------------------------------------------------------------------------- gradients that would be lost
def test_a_tangent_is_refused_like_a_gradient(dev):
    """Forward-mode differentiation: a dual tensor does not require a gradient, and its tangent would be dropped."""
    x = torch.ones(8, 4, 64, device=dev)
    starts = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    freq, pos = acnative.rotary_frequencies(64, device=dev), torch.zeros(8, dtype=torch.int32, device=dev)
    w = torch.ones(64, device=dev)
    mean = torch.zeros(8, 4, device=dev)
    fwd = torch.autograd.forward_ad
    calls = (lambda t: acnative.rotary(t, None, pos, freq), lambda t: acnative.rotary(x, t, pos, freq), lambda t: acnative.rotary(x, None, pos, freq, out_q=t),
             lambda t: acnative.attention_packed(t, x, x, starts), lambda t: acnative.attention_packed(x, t, x, starts),
             lambda t: acnative.attention_packed(x, x, t, starts), lambda t: acnative.layer_norm(t), lambda t: acnative.layer_norm(x, out=t),
             lambda t: acnative.layer_norm_backward(t, x, None, mean, mean), lambda t: acnative.layer_norm_backward(x, t, None, mean, mean))
    vectors = (lambda t: acnative.layer_norm(x, t), lambda t: acnative.layer_norm(x, w, t), lambda t: acnative.layer_norm_backward(x, x, t, mean, mean))
    with fwd.dual_level():
        for call in calls:
            with pytest.raises(RuntimeError, match="gradient"):
                call(fwd.make_dual(torch.ones_like(x), torch.ones_like(x)))
            call(torch.ones_like(x))                              # without a tangent: fine inside a level too
        for call in vectors:
            with pytest.raises(RuntimeError, match="gradient"):
                call(fwd.make_dual(w.clone(), torch.ones_like(w)))
        with pytest.raises(RuntimeError, match="gradient"):
            acnative.rotary(x, None, pos, fwd.make_dual(freq.clone(), torch.ones_like(freq)))


def test_frequencies_and_statistics_that_require_a_gradient_are_refused(dev):
    x = torch.ones(8, 4, 64, device=dev)
    pos, freq = torch.zeros(8, dtype=torch.int32, device=dev), acnative.rotary_frequencies(64, device=dev)
    stat = torch.ones(8, 4, device=dev)
    learned = freq.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        acnative.rotary(x, None, pos, learned)
    for a, b in ((stat.clone().requires_grad_(), stat), (stat, stat.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="gradient"):
            acnative.layer_norm_backward(x, x, None, a, b)
    with torch.no_grad():
        assert acnative.rotary(x, None, pos, learned).shape == x.shape


# ------------------------------------------------------------------------------------------------ norm beside its input
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_layer_norm_into_the_other_columns_of_its_rows(dev, kind):
    """x and out as column ranges of one buffer: their spans cross, their entries do not."""
    T, C = 33, 96
    both = torch.cat([_randn((T, C), 1, kind), torch.full((T, C), 7.0, dtype=KINDS[kind])], 1).to(dev)
    x, out = both[:, :C], both[:, C:]
    w, b = _randn((C,), 2, kind).to(dev), _randn((C,), 3, kind).to(dev)
    want = acnative.layer_norm(x.contiguous(), w, b)
    assert acnative.layer_norm(x, w, b, out=out) is out
    assert torch.equal(out, want) and torch.equal(x.cpu(), _randn((T, C), 1, kind))
    three = both.view(3, 11, 2 * C)
    assert torch.equal(acnative.layer_norm(three[..., C:], w, b, out=three[..., :C]).reshape(T, C), acnative.layer_norm(want, w, b))
    for bad in (both[:, 1:C + 1], both[:, C - 1:2 * C - 1]):
        with pytest.raises(ValueError, match="overlaps"):
            acnative.layer_norm(both[:, :C], w, b, out=bad)


def test_writing_into_a_tensor_is_seen_by_autograd(dev):
    """A tensor that a graph has saved and an operator then writes into: backward has to refuse, not to use the new values."""
    pos, freq = torch.arange(8, dtype=torch.int32, device=dev), acnative.rotary_frequencies(64, device=dev)
    starts = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    other = torch.ones(8, 4, 64, device=dev)
    for write in (lambda t: acnative.rotary(t, None, pos, freq, out_q=t), lambda t: acnative.rotary(other, t, pos, freq, out_k=t),
                  lambda t: acnative.layer_norm(t, out=t), lambda t: acnative.attention_packed(other, other, other, starts, out=t)):
        leaf = torch.ones(8, 4, 64, device=dev, requires_grad=True)
        y = leaf * 2
        z = (y * y).sum()
        write(y.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    with torch.inference_mode():
        t = torch.ones(8, 4, 64, device=dev)
        assert acnative.rotary(t, None, pos, freq, out_q=t) is t


# --------------------------------------------------------------------------- attention on values at the ends of a type
def _lagging(n, keys, H, G, D, kind, seed):
    """q and k whose first 32 keys score about 0 and the later ones up to 2^7.5 times their weight: the running maximum stays."""
    q, k = torch.zeros(n, H, D), torch.zeros(keys, G, D)
    q[..., 0] = 1.0
    k[:, :, 0] = 7.4 * math.log(2.0) * D ** 0.5 * (0.9 + 0.1 * torch.rand(keys, G, generator=torch.Generator().manual_seed(seed)))
    k[:32, :, 0] = 0.01
    q[..., 1:], k[..., 1:] = 0.05 * _randn((n, H, D - 1), seed, "fp32"), 0.05 * _randn((keys, G, D - 1), seed + 1, "fp32")
    return q.to(KINDS[kind]), k.to(KINDS[kind])


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("H,G,D,queries,keys,causal", [(2, 2, 64, [300], [300], False), (2, 1, 128, [200, 70], [500, 70], True), (8, 2, 64, [1, 1], [3000, 700], False),
                                                       (2, 2, 80, [150], [150], True), (4, 1, 128, [1, 3], [5000, 64], True)])
def test_attention_of_values_near_the_largest(dev, kind, H, G, D, queries, keys, causal):
    """Finite values whose weighted sum leaves the type's range where their weighted mean does not."""
    sq, sk = _starts(queries), _starts(keys)
    q, k = _lagging(int(sq[-1]), int(sk[-1]), H, G, D, kind, D)
    v = (_randn((int(sk[-1]), G, D), 9, "fp32").clamp(-4, 4) * 8e37).to(KINDS[kind])
    ref = opacked.attention(q, k, v, sq, sk, causal)
    got, sums = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), sk.to(dev), max_q=max(queries), max_k=max(keys), causal=causal,
                                          want_sums=True)
    assert torch.isfinite(got).all()
    _check_attention(got, sums, ref, kind, D, "near the largest")


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("queries,keys", [([90], [90]), ([1], [3000]), ([300, 20], [400, 20])])
def test_attention_infinite_values_of_small_weight(dev, kind, queries, keys):
    """An infinite value that a row sees passes however little it weighs: 2^-50 is nothing in fp16, and 0 times infinity would be NaN."""
    H, D = 2, 64
    sq, sk = _starts(queries), _starts(keys)
    q, k, v = torch.zeros(int(sq[-1]), H, D), torch.zeros(int(sk[-1]), H, D), _randn((int(sk[-1]), H, D), 3, kind)
    q[..., 0] = 1.0
    k[..., 0] = 0.1 * _randn((int(sk[-1]), H), 4, "fp32")
    k[40, 0, 0] = -50 * math.log(2.0) * 8.0
    v[40, 0, 5], v[40, 0, 6] = math.inf, -math.inf
    q, k = q.to(KINDS[kind]), k.to(KINDS[kind])
    ref = opacked.attention(q, k, v, sq, sk, False)
    assert (ref["out"][:queries[0], 0, 5] == math.inf).all() and (ref["out"][:queries[0], 0, 6] == -math.inf).all()
    got, sums = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), sk.to(dev), max_q=max(queries), max_k=max(keys), want_sums=True)
    _check_attention(got, sums, ref, kind, D, "small weight")


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("queries,keys", [([90], [96]), ([1], [3000]), ([300, 20], [416, 32])])
def test_attention_of_a_bad_value_that_every_row_sees(dev, kind, bad, queries, keys):
    """It makes its own column of its own head NaN (or infinite) and touches no other."""
    H, D = 2, 80
    sq, sk = _starts(queries), _starts(keys)
    q, k, v = (_randn((n, H, D), i, kind) for i, n in enumerate((int(sq[-1]), int(sk[-1]), int(sk[-1]))))
    v[17, 1, 70] = bad
    ref = opacked.attention(q, k, v, sq, sk, False)
    assert not torch.isfinite(ref["out"][:queries[0], 1, 70]).any() and (~torch.isfinite(ref["out"])).sum() == queries[0]
    got, sums = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), sk.to(dev), max_q=max(queries), max_k=max(keys), want_sums=True)
    _check_attention(got, sums, ref, kind, D, "bad value")


# --------------------------------------------------------------------------------- attention's plans for many rows
def _plan(dev, kind, heads, kv_heads, D, queries):
    """The rule of make_plan (csrc/attention.hip) for 16-bit rows: 2: 32 rows and split keys, 1: 128 rows, 0: 256 rows (64 to a wave),
    3: 128 rows (64 to a wave, two waves)."""
    cus = torch.cuda.get_device_properties(dev).multi_processor_count
    rows, pairs, tokens = max(max(queries), -(-sum(queries) // len(queries))) * (heads // kv_heads), len(queries) * kv_heads, sum(queries)
    if rows <= 32:
        return 2
    if kind == "fp32" or D * 2 > 256 or pairs * -(-rows // 256) < 2 * cus:
        return 1
    return 3 if D * 2 > 128 and tokens * heads // 256 < 8 * cus else 0


def _many(count, top, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, top, (count,), generator=g).tolist()
    n[:14] = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257]
    n[20] = 300
    return n


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("plan,D,heads,kv_heads", [(0, 8, 8, 4), (0, 24, 8, 4), (0, 32, 4, 4), (0, 48, 8, 4), (0, 64, 12, 4), (0, 64, 4, 4),
                                                   (3, 72, 8, 4), (3, 80, 4, 4), (3, 96, 8, 4), (3, 104, 4, 4), (3, 128, 12, 4), (3, 128, 4, 4)])
def test_attention_of_many_rows(dev, kind, plan, D, heads, kv_heads):
    """64 rows a wave: masks over two blocks of rows, shared heads, keys of other lengths, log-sums, ends inside tiles."""
    queries, keys = _many(70 if heads > kv_heads else 132, 120, D), _many(70 if heads > kv_heads else 132, 160, D + 1)
    assert _plan(dev, kind, heads, kv_heads, D, queries) == plan
    _run(dev, kind, heads, kv_heads, D, queries, causal=D % 16 == 0, seed=D)
    keys[1:14] = [400, 0, 32, 20, 330, 64, 10, 300, 128, 129, 1, 500, 257]
    _run(dev, kind, heads, kv_heads, D, queries, keys, causal=True, seed=D + 1)
    if D in (64, 80, 128):
        _run(dev, kind, heads, kv_heads, D, queries, keys, causal=False, seed=D + 2, qscale=40.0, scale=-0.1, before=3, behind=5)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [80, 128])
def test_attention_of_many_rows_of_wide_heads(dev, kind, D):
    """Heads of more than 128 bytes in blocks of 256 rows: 2^19 rows or more."""
    g = torch.Generator().manual_seed(D)
    queries = torch.randint(20, 60, (430,), generator=g).tolist() + [300, 257, 64, 1, 0]
    assert _plan(dev, kind, 32, 8, D, queries) == 0
    _run(dev, kind, 32, 8, D, queries, causal=True, seed=D)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("plan,D", [(0, 64), (0, 40), (3, 72), (3, 128)])
def test_attention_of_many_rows_what_a_row_does_not_see_cannot_touch_it(dev, kind, plan, D):
    """Infinities and NaN in keys and values behind a causal row, in the next sequence and in the next head, with 64 rows a wave."""
    n, H = 150, 8
    lengths = [n, 40] + _many(68, 60, D)
    lengths[22] = 200
    assert _plan(dev, kind, H, H, D, lengths) == plan
    sq = _starts(lengths, 3)
    T = int(sq[-1]) + 5
    q, k, v = (_randn((T, H, D), i, kind) for i in (1, 2, 3))
    for t in (k, v):
        t[:3] = math.nan
        t[int(sq[-1]):] = math.inf
    v[3 + 100, 0, 5] = math.inf
    v[3 + 120, 0, 6] = math.nan
    v[3 + 130, 1, 7] = -math.inf
    k[3 + 140, 0] = math.nan
    clean = k.clone()
    clean[3 + 140, 0] = 0.0
    ref = opacked.attention(q, clean, v, sq, sq, True)
    ref["out"][3 + 140:3 + n, 0] = math.nan                        # these rows see the NaN key: NaN throughout
    out = torch.full((T, H, D), 7.0, dtype=KINDS[kind], device=dev)
    acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), max_q=max(lengths), max_k=max(lengths), causal=True, out=out)
    assert (out[:3] == 7.0).all() and (out[int(sq[-1]):] == 7.0).all()
    inside = slice(3, int(sq[-1]))
    _check_attention(out[inside], None, {key: x[inside] for key, x in ref.items()}, kind, D, "poisoned")
