"""CPU: what the packed-sequence operators refuse, before anything is launched, and their host-side helpers."""
import ctypes
import math

import pytest
import torch

import acnative
from oracle import packed as opacked


def _rotary(**over):
    a = acnative.RotaryArgs()
    a.src[0], a.dst[0], a.src[1], a.dst[1] = 4096, 8192, 0, 0
    a.heads[0], a.heads[1], a.src_token[0], a.src_head[0], a.dst_token[0], a.dst_head[0] = 2, 0, 128, 64, 128, 64
    a.positions, a.position_axis, a.frequencies, a.tokens, a.type, a.layout = 4096, 4, 4096, 4, 2, 0
    a.dim, a.part, a.offset, a.axes, a.inverse, a.amplitude = 64, 64, 0, 1, 0, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [({"type": 5}, "unknown type"), ({"layout": 2}, "unknown layout"), ({"dim": 2000, "part": 2}, "head dim"),
                                       ({"part": 63}, "multiple of 2"), ({"part": 62, "axes": 2}, "multiple of 2"), ({"part": 0}, "multiple of 2"),
                                       ({"offset": 2}, "outside a head"), ({"offset": -1, "part": 2}, "outside a head"), ({"tokens": -1}, "counts"),
                                       ({"frequencies": 0}, "null"), ({"frequencies": 4100}, "misaligned"), ({"positions": 4098}, "misaligned"),
                                       ({"layout": 1, "offset": 1, "part": 2}, "even")])
def test_rotary_refuses(over, text):
    lib = acnative.lib()
    assert lib.ac_rotary(ctypes.byref(_rotary(**over)), None) == 1
    assert text in lib.ac_last_error().decode()


def test_rotary_of_no_token_is_fine():
    assert acnative.lib().ac_rotary(ctypes.byref(_rotary(tokens=0)), None) == 0


def _attention(**over):
    a = acnative.AttentionArgs()
    a.q = a.k = a.v = a.out = a.starts_q = a.starts_k = 4096
    a.q_token = a.k_token = a.v_token = a.out_token = 128
    a.q_head = a.k_head = a.v_head = a.out_head = 64
    a.tokens_q = a.tokens_k = 100
    a.sequences, a.heads, a.kv_heads, a.dim, a.max_q, a.max_k, a.causal, a.type, a.scale = 2, 2, 2, 64, 50, 50, 0, 2, 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [({"type": 3}, "unknown type"), ({"heads": 3}, "cannot share"), ({"kv_heads": 0}, "cannot share"), ({"dim": 60}, "head dim"),
                                       ({"dim": 264}, "head dim"), ({"dim": 0}, "head dim"), ({"sequences": -1}, "negative"), ({"q": 0}, "null"), ({"v": 0}, "null"),
                                       ({"starts_k": 0}, "null"), ({"k": 4104}, "aligned"), ({"q_token": 130}, "strides"), ({"out_head": -64}, "strides"),
                                       ({"k_token": 1 << 20}, "stride"), ({"tokens_q": 1 << 31}, "too many tokens"), ({"tokens_k": 1 << 31}, "too many tokens"),
                                       ({"scale": math.inf}, "finite"), ({"scale": math.nan}, "finite")])
def test_attention_refuses(over, text):
    lib = acnative.lib()
    assert lib.ac_attention_packed(ctypes.byref(_attention(**over)), None, 0, None) == 1
    assert text in lib.ac_last_error().decode()


def test_attention_workspace():
    """Needed where few rows meet long keys, and asked for by name when it is missing."""
    lib = acnative.lib()
    assert lib.ac_attention_packed_workspace_bytes(ctypes.byref(_attention())) == 0
    long = _attention(tokens_q=2, tokens_k=100000, max_q=1, max_k=50000)
    n = lib.ac_attention_packed_workspace_bytes(ctypes.byref(long))
    assert n > 2 * 2 * 64 * 4
    assert lib.ac_attention_packed(ctypes.byref(long), None, 0, None) == 2 and b"workspace" in lib.ac_last_error()
    assert lib.ac_attention_packed(ctypes.byref(long), 4096, n - 1, None) == 2
    assert lib.ac_attention_packed(ctypes.byref(_attention(tokens_q=0)), None, 0, None) == 0
    assert lib.ac_attention_packed(ctypes.byref(_attention(sequences=0)), None, 0, None) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 2, 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        acnative.rotary(x, None, torch.zeros(4, dtype=torch.int32), torch.zeros(32, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        acnative.attention_packed(x, x, x, torch.zeros(2, dtype=torch.int32))


def test_overlap_checks():
    base = torch.zeros(10, 8, 16)
    q, k = base[:, :4], base[:, 4:6]
    assert acnative._apart(q, k) and acnative._apart(k, q) and not acnative._apart(q, base[:, 3:5]) and not acnative._apart(q, q)
    assert acnative._apart(base[:5], base[5:]) and not acnative._apart(base[:6], base[5:])
    assert not acnative._apart(q, base[1:, :4].transpose(0, 1))
    assert acnative._same_view(q, base[:, :4]) and not acnative._same_view(q, base[:, 1:5])
    acnative._writable(base[:, 2:, 3:], "out")
    acnative._writable(base.transpose(0, 1), "out")
    for bad in (base[:, :1].expand(10, 4, 16), base.as_strided((10, 8, 16), (16, 16, 1))):
        with pytest.raises(ValueError, match="overlap"):
            acnative._writable(bad, "out")


def test_helpers():
    starts, longest = acnative.sequence_starts([3, 0, 7], "cpu")
    assert starts.tolist() == [0, 3, 3, 10] and starts.dtype == torch.int32 and longest == 7
    assert acnative.sequence_starts([], "cpu")[0].tolist() == [0]
    with pytest.raises(ValueError):
        acnative.sequence_starts([3, -1], "cpu")
    with pytest.raises(ValueError):
        acnative.sequence_starts([1 << 30, 1 << 30], "cpu")
    for bad in ({"part": 7}, {"part": 6, "axes": 2}, {"part": 8, "base": 0.0}, {"part": 8, "factor": -1.0}, {"part": 8, "low": 3.0, "high": 3.0}):
        with pytest.raises(ValueError):
            acnative.rotary_frequencies(**bad)
    f = acnative.rotary_frequencies(32, 10000.0, factor=4.0, original=2048)
    assert torch.allclose(f, opacked.frequencies(32, 10000.0, 1, 4.0, 2048), rtol=1e-14, atol=0)
    assert f[0, 0] == 1.0 and abs(f[0, -1].item() - 10000.0 ** (-15 / 16) / 4) < 1e-18


def test_oracle_against_itself():
    """The oracle's attention on one unmasked sequence is a plain softmax, and its mask leaves rows empty where it should."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(6, 2, 8, generator=g, dtype=torch.float64) for _ in range(3))
    r = opacked.attention(q, k, v, [0, 6], [0, 6], False)
    p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(8), -1)
    assert torch.allclose(r["out"], torch.einsum("hij,jhd->ihd", p, v))
    r = opacked.attention(q, k[:2], v[:2], [0, 6], [0, 2], True)
    assert (r["out"][:4] == 0).all() and (r["sums"][:4] == -math.inf).all() and torch.allclose(r["out"][4], v[0])


def _norm(**over):
    a = acnative.NormArgs()
    a.x = a.y = a.dy = a.dx = a.weight = a.bias = 4096
    a.mean = a.rstd = 4096
    a.x_row = a.y_row = a.dy_row = a.dx_row = 64
    a.rows, a.width, a.type, a.weight_type, a.eps = 4, 64, 2, 0, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [({"type": 7}, "unknown type"), ({"weight_type": 1}, "weights"), ({"rows": -1}, "rows"), ({"rows": 1 << 31}, "rows"),
                                       ({"width": 0}, "width"), ({"width": (1 << 20) + 1}, "width"), ({"x": 0}, "null"), ({"y": 0}, "null"),
                                       ({"mean": 0}, "together"), ({"x": 4097}, "misaligned"), ({"weight": 4098}, "misaligned")])
def test_layer_norm_refuses(over, text):
    lib = acnative.lib()
    assert lib.ac_layer_norm(ctypes.byref(_norm(**over)), None) == 1
    assert text in lib.ac_last_error().decode()


def test_layer_norm_backward_refuses_and_asks_for_its_workspace():
    lib = acnative.lib()
    for over, text in (({"dy": 0}, "null"), ({"mean": 0}, "null"), ({"dx": 4097}, "misaligned"), ({"dweight": 4098}, "misaligned"), ({"width": 0}, "width")):
        assert lib.ac_layer_norm_backward(ctypes.byref(_norm(**over)), None, 0, None) == 1
        assert text in lib.ac_last_error().decode()
    n = lib.ac_layer_norm_backward_workspace_bytes(ctypes.byref(_norm(dweight=4096)))
    assert n >= 2 * 64 * 4 and lib.ac_layer_norm_backward_workspace_bytes(ctypes.byref(_norm())) == 0
    assert lib.ac_layer_norm_backward(ctypes.byref(_norm(dweight=4096)), 4096, n - 1, None) == 2 and b"workspace" in lib.ac_last_error()
    assert lib.ac_layer_norm_backward(ctypes.byref(_norm(dx=0)), None, 0, None) == 0      # nothing wanted
    assert lib.ac_layer_norm(ctypes.byref(_norm(rows=0)), None) == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        acnative.layer_norm(torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        acnative.layer_norm_backward(torch.zeros(4, 8), torch.zeros(4, 8), None, torch.zeros(4), torch.zeros(4))


def test_attention_refuses_more_pairs_than_a_launch_takes():
    lib = acnative.lib()
    assert lib.ac_attention_packed(ctypes.byref(_attention(sequences=1 << 20)), None, 0, None) == 1      # two key heads
    assert "too many sequences" in lib.ac_last_error().decode()
    assert lib.ac_attention_packed_workspace_bytes(ctypes.byref(_attention(sequences=1 << 20))) == 0


@pytest.mark.parametrize("over,text", [({"offset": (1 << 31) - 2, "part": 2}, "outside a head"), ({"offset": (1 << 31) - 64}, "outside a head"),
                                       ({"part": (1 << 31) - 2, "offset": 2}, "outside a head"), ({"axes": (1 << 31) - 1}, "multiple of 2"),
                                       ({"axes": 1 << 30}, "multiple of 2"), ({"axes": (1 << 30) + 16}, "multiple of 2"), ({"axes": -1}, "multiple of 2")])
def test_rotary_refuses_what_only_32_bits_would_let_through(over, text):
    """offset + part and 2 * axes, formed in 32 bits, wrap around to values that pass."""
    lib = acnative.lib()
    assert lib.ac_rotary(ctypes.byref(_rotary(**over)), None) == 1
    assert text in lib.ac_last_error().decode()


@pytest.mark.parametrize("over", [{"tokens_q": 1 << 62, "heads": 4, "kv_heads": 1}, {"tokens_k": (1 << 63) - 1}, {"tokens_q": (1 << 63) - 1, "heads": 2, "kv_heads": 1}])
def test_attention_refuses_what_only_64_bits_would_let_through(over):
    """tokens_q * heads and tokens_k + a tile, formed in 64 bits, wrap around to values that pass."""
    lib = acnative.lib()
    assert lib.ac_attention_packed(ctypes.byref(_attention(**over)), None, 0, None) == 1
    assert "too many tokens" in lib.ac_last_error().decode()
    assert lib.ac_attention_packed_workspace_bytes(ctypes.byref(_attention(**over))) == 0
