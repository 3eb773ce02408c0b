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
