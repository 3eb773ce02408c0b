"""GPU parity: rotary positions and attention over packed sequences against the float64 oracle (oracle/packed.py).

Error bounds, per entry.  u = half a step of the tensor's type (eps / 2), e = 2^-24 (half a step of fp32).
rotary     the factors are right to 2^-22 of their own (a fp32 polynomial of a fp64 remainder), two products and a sum in
           fp32 on top: (2^-22 + 4 e) m (|a| + |b|), and the result's rounding u |out|.
attention  scores: D products summed in fp32 in an order that is not ours (2 D e of the sum of magnitudes S), scaled and
           shifted in the log2 domain (6 e S): es = (2 D + 6) e S.  A weight is off by 2 es + 4 e relative to the row's (its own and the
           total's error, the exponential's), by n e for the sums over n keys, and by u where it is rounded for the matrix
           product (16-bit types; fp16 weights under 2^-14 lose 2^-25 of the row's largest): (2 es + (n + 8) e + u) sum p |v| +
           [fp16] 2^-25 sum |v|, and the result's rounding u |out|.
           log-sums: es + (n + 8) e + 2 e |sum|.
"""
import math

import pytest
import torch

import acnative
from oracle import packed as opacked

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
KINDS = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _u(kind):
    return torch.finfo(KINDS[kind]).eps / 2


def _randn(shape, seed, kind, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(KINDS[kind])


def _starts(lengths, before=0):
    out = [before]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def _check_attention(got, sums, ref, kind, D, what=""):
    u = _u(kind)
    es = (2 * D + 6) * E * ref["score"]
    tol = u * ref["out"].abs() + (2 * es + (ref["keys"] + 8) * E + (u if kind != "fp32" else 0.0))[..., None] * ref["weighted"] + 1e-30
    if kind == "fp16":
        tol = tol + 2.0 ** -25 * ref["plain"] + 2.0 ** -25          # weights and results under the smallest normal number
    got = got.cpu().double()
    odd = ~torch.isfinite(ref["out"])
    assert torch.equal(torch.isnan(got), torch.isnan(ref["out"])), what
    assert torch.equal(got[torch.isinf(ref["out"])], ref["out"][torch.isinf(ref["out"])]), what
    err = torch.where(odd, torch.zeros_like(got), (got - ref["out"]).abs())
    worst = (err / tol)[~odd].max().item() if (~odd).any() else 0.0
    assert worst <= 1.0, "%s: error %.3g of its bound" % (what, worst)
    if sums is not None:
        s = sums.cpu().double()
        none = torch.isinf(ref["sums"])
        assert torch.equal(s[none], ref["sums"][none]), what
        bound = es + (ref["keys"] + 8) * E + 2 * E * ref["sums"].abs()
        assert ((s - ref["sums"]).abs()[~none] <= bound[~none]).all(), what
    return worst


def _run(dev, kind, heads, kv_heads, D, queries, keys=None, causal=False, seed=0, scale=None, sums=True, hints=True, qscale=1.5, before=0, behind=0):
    sq = _starts(queries, before)
    sk = sq if keys is None else _starts(keys, before)
    Tq, Tk = int(sq[-1]) + behind, int(sk[-1]) + behind
    q, k, v = (_randn((T, H, D), seed + i, kind, s) for i, (T, H, s) in enumerate(((Tq, heads, qscale), (Tk, kv_heads, 1.0), (Tk, kv_heads, 1.0))))
    ref = opacked.attention(q, k, v, sq, sk, causal, scale)
    more = {"max_q": max(queries), "max_k": max(keys or queries)} if hints else {}
    got = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), sk.to(dev), causal=causal, scale=scale, want_sums=sums, **more)
    got, s = got if sums else (got, None)
    return _check_attention(got, s, ref, kind, D, "%s %d/%d heads of %d, %s x %s%s" % (kind, heads, kv_heads, D, queries, keys, " causal" if causal else ""))


# ----------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,G,D,part,offset,axes", [(1, 1, 1, 64, 64, 0, 1), (17, 12, 12, 64, 64, 0, 2), (301, 4, 2, 80, 24, 8, 1), (5, 3, 1, 36, 20, 6, 1),
                                                      (130, 32, 8, 128, 64, 64, 1), (3, 2, 2, 256, 256, 0, 2), (9, 5, 1, 1024, 1024, 0, 1), (40, 1, 1, 2, 2, 0, 1)])
def test_rotary(dev, kind, layout, T, H, G, D, part, offset, axes):
    q, k = _randn((T, H, D), 1, kind), _randn((T, G, D), 2, kind)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(-5, 4_000_000 if axes == 1 else 300, (axes, T), generator=g, dtype=torch.int32)
    freq = acnative.rotary_frequencies(part, 10000.0, axes=axes)
    got = acnative.rotary(q.to(dev), k.to(dev), pos.to(dev), freq.to(dev), layout=layout, offset=offset, amplitude=1.25)
    for x, y in zip((q, k), got):
        ref, size = opacked.rotary(x, pos, freq, layout, offset, 1.25)
        tol = _u(kind) * ref.abs() + (2.0 ** -22 + 4 * E) * size + (2.0 ** -25 if kind == "fp16" else 0.0)
        assert ((y.cpu().double() - ref).abs() <= tol).all()
        rest = torch.ones(D, dtype=torch.bool)
        rest[offset:offset + part] = False
        assert torch.equal(y.cpu()[..., rest], x[..., rest])


def test_rotary_in_place_on_slices_and_back(dev):
    """q and k as slices of one projection's rows, turned in place; v stays; turned back they are what they were, to rounding."""
    T, H, G, D = 77, 6, 2, 64
    qkv = _randn((T, H + 2 * G, D), 5, "fp32").to(dev)
    before = qkv.clone()
    q, k = qkv[:, :H], qkv[:, H:H + G]
    pos = torch.arange(T, dtype=torch.int64, device=dev) * 1000
    freq = acnative.rotary_frequencies(D, device=dev)
    out = acnative.rotary(q, k, pos, freq, out_q=q, out_k=k)
    assert out[0] is q and out[1] is k
    assert torch.equal(qkv[:, H + G:], before[:, H + G:])
    ref, _ = opacked.rotary(before[:, :H].cpu(), pos.cpu(), freq.cpu(), "half", 0, 1.0)
    assert (q.cpu().double() - ref).abs().max() < 1e-5
    acnative.rotary(q, k, pos, freq, out_q=q, out_k=k, inverse=True)
    assert (qkv - before).abs().max() < 1e-5


@pytest.mark.parametrize("strides", ["odd", "expanded", "transposed"])
def test_rotary_strides(dev, strides):
    T, H, D = 19, 4, 48
    base = _randn((T + 1, H + 1, D + 3), 7, "bf16")
    x = base[1:, 1:, 3:] if strides == "odd" else base[:T, :1, :D].expand(T, H, D) if strides == "expanded" else base[:H, :H, :D].transpose(0, 1)
    T = x.shape[0]
    pos = torch.arange(T, dtype=torch.int32)
    freq = acnative.rotary_frequencies(D)
    dx = base.to(dev)
    dx = dx[1:, 1:, 3:] if strides == "odd" else dx[:T, :1, :D].expand(T, H, D) if strides == "expanded" else dx[:H, :H, :D].transpose(0, 1)
    got = acnative.rotary(dx, None, pos.to(dev), freq.to(dev))
    ref, size = opacked.rotary(x, pos, freq, "half", 0, 1.0)
    assert ((got.cpu().double() - ref).abs() <= _u("bf16") * ref.abs() + (2.0 ** -22 + 4 * E) * size).all()


@pytest.mark.parametrize("factor,original", [(1.0, None), (8.0, None), (8.0, 4096), (0.5, 100)])
def test_rotary_frequencies(dev, factor, original):
    got = acnative.rotary_frequencies(64, 5000.0, axes=2, factor=factor, original=original, device=dev)
    ref = opacked.frequencies(64, 5000.0, 2, factor, original)
    assert got.shape == (2, 16) and got.dtype == torch.float64
    assert ((got.cpu() - ref).abs() <= 1e-14 * ref).all()


# -------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 64, 72, 80, 96, 104, 128, 144, 160, 176, 192, 224, 256])
def test_attention_head_dims(dev, kind, D):
    _run(dev, kind, 2, 1, D, [70, 1, 0, 33], causal=True, seed=D)
    _run(dev, kind, 2, 2, D, [40, 300], causal=False, seed=D + 1)
    _run(dev, kind, 4, 1, D, [1, 3], [200, 77], causal=True, seed=D + 2)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys", [([1], None), ([2, 1, 1], None), ([31, 32, 33, 63, 64, 65], None), ([127, 129, 255, 257], None), ([0, 5, 0, 0, 9], None),
                                          ([785, 197], None), ([5, 60, 1, 0], [300, 60, 1000, 40]), ([70, 200, 1, 3], [10, 0, 0, 2]), ([600], [90]), ([513], [1025])])
def test_attention_lengths(dev, kind, causal, queries, keys):
    _run(dev, kind, 3, 3, 64, queries, keys, causal, seed=len(queries))
    _run(dev, kind, 8, 2, 128, queries, keys, causal, seed=len(queries) + 7)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (5, 1), (6, 2), (32, 1), (40, 1), (7, 7), (21, 3)])
def test_attention_grouped_heads(dev, kind, heads, kv_heads):
    _run(dev, kind, heads, kv_heads, 64, [45, 1, 130], causal=True, seed=heads)
    _run(dev, kind, heads, kv_heads, 64, [1, 1, 1], [5, 700, 64], causal=True, seed=heads + 1)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_attention_single_queries_on_long_keys(dev, kind):
    """The key axis is split and joined; a sequence without keys, one with a single key, ends inside a tile."""
    _run(dev, kind, 8, 2, 128, [1] * 6, [5000, 1, 0, 512, 513, 3333], causal=True, seed=1)
    _run(dev, kind, 4, 4, 64, [2, 1, 3], [4000, 2047, 1], causal=False, seed=2)
    _run(dev, kind, 2, 1, 256, [1, 9], [2500, 1100], causal=True, seed=3)
    _run(dev, kind, 2, 2, 80, [300], [4100], causal=True, seed=4)


def test_attention_hints_do_not_matter(dev):
    """Too small, too large and missing bounds of the lengths: the same rows."""
    sq, sk = _starts([1, 700, 3]), _starts([900, 700, 4000])
    q, k, v = _randn((704, 4, 64), 1, "bf16"), _randn((5600, 2, 64), 2, "bf16"), _randn((5600, 2, 64), 3, "bf16")
    ref = opacked.attention(q, k, v, sq, sk, True)
    args = [t.to(dev) for t in (q, k, v, sq, sk)]
    for max_q, max_k in ((None, None), (1, 1), (1, 100000), (700, 10), (0, 0), (10 ** 6, 10 ** 6), (100, 4000)):
        got, sums = acnative.attention_packed(*args, max_q=max_q, max_k=max_k, causal=True, want_sums=True)
        _check_attention(got, sums, ref, "bf16", 64, "max_q=%s max_k=%s" % (max_q, max_k))


def test_attention_extremes(dev):
    """A late key far ahead of the rest, scores in the hundreds, equal scores, a scale of zero and a negative one."""
    _run(dev, "bf16", 2, 2, 64, [300], causal=False, seed=3, qscale=60.0)
    _run(dev, "fp16", 2, 1, 128, [257], causal=True, seed=4, qscale=60.0)
    _run(dev, "fp32", 2, 1, 64, [257], causal=True, seed=5, qscale=60.0)
    for kind in ("fp32", "fp16", "bf16"):
        _run(dev, kind, 2, 2, 64, [100, 3], causal=True, seed=6, scale=0.0)
        _run(dev, kind, 2, 2, 64, [100, 3], causal=True, seed=7, scale=-0.2)
        sq = _starts([400])
        q, k, v = torch.ones(400, 1, 64), _randn((400, 1, 64), 8, "fp32"), _randn((400, 1, 64), 9, "fp32")
        k = k * 0.01
        k[390] = 8.0                                               # one key takes nearly everything, late
        q, k, v = (t.to(KINDS[kind]) for t in (q, k, v))
        got, sums = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), want_sums=True)
        _check_attention(got, sums, opacked.attention(q, k, v, sq, sq, False), kind, 64, "late maximum")


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 72])
def test_attention_what_a_row_does_not_see_cannot_touch_it(dev, kind, D):
    """Infinities and NaN in keys and values behind a causal row, behind a sequence, and in the next head."""
    n, H = 150, 2
    sq = _starts([n, 40], 3)
    T = int(sq[-1]) + 5
    q, k, v = (_randn((T, H, D), i, kind) for i in (1, 2, 3))
    for t in (k, v):
        t[:3] = math.nan                                           # before the first sequence
        t[int(sq[-1]):] = math.inf                                 # behind the last
    v[3 + 100, 0, 5] = math.inf
    v[3 + 120, 0, 6] = math.nan
    v[3 + 130, 1, 7] = -math.inf
    k[3 + 140, 0] = math.nan
    ref = opacked.attention(q, k, v, sq, sq, True)
    clean = k.clone()
    clean[3 + 140, 0] = 0.0
    seen_bad = torch.zeros(T, H, dtype=torch.bool)
    seen_bad[3 + 140:3 + n, 0] = True                              # these rows see the NaN key: NaN throughout
    ref = opacked.attention(q, clean, v, sq, sq, True)
    ref["out"][seen_bad] = math.nan
    out = torch.full((T, H, D), 7.0, dtype=KINDS[kind], device=dev)
    got = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), causal=True, out=out)
    assert got is out
    assert (got[:3] == 7.0).all() and (got[int(sq[-1]):] == 7.0).all()
    inside = slice(3, int(sq[-1]))
    for key in ref:
        ref[key] = ref[key][inside]
    _check_attention(got[inside], None, ref, kind, D, "poisoned")


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_attention_rows_outside_the_sequences(dev, kind):
    sq = _starts([20, 0, 30], 4)
    T = int(sq[-1]) + 6
    q, k, v = (_randn((T, 4, 64), i, kind).to(dev) for i in (1, 2, 3))
    fresh, sums = acnative.attention_packed(q, k, v, sq.to(dev), want_sums=True)
    for rows in (slice(0, 4), slice(T - 6, T)):
        assert (fresh[rows] == 0).all() and (sums[rows] == -math.inf).all()
    kept = torch.full_like(fresh, 3.0)
    acnative.attention_packed(q, k, v, sq.to(dev), out=kept)
    assert (kept[:4] == 3.0).all() and (kept[T - 6:] == 3.0).all() and torch.equal(kept[4:T - 6], fresh[4:T - 6])
    none = acnative.attention_packed(q, k, v, torch.zeros(1, dtype=torch.int32, device=dev))
    assert (none == 0).all()
    empty = acnative.attention_packed(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=dev))
    assert empty.shape == (0, 4, 64)
    nokeys = acnative.attention_packed(q, k[:0], v[:0], sq.to(dev), torch.zeros(4, dtype=torch.int32, device=dev))
    assert (nokeys == 0).all()


def test_attention_starts_out_of_range_are_clamped(dev):
    q, k, v = (_randn((50, 2, 64), i, "bf16") for i in (1, 2, 3))
    wild = torch.tensor([-7, 20, 90], dtype=torch.int32)
    tame = torch.tensor([0, 20, 50], dtype=torch.int32)
    ref = opacked.attention(q, k, v, tame, tame, False)
    got, sums = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), wild.to(dev), want_sums=True)
    _check_attention(got, sums, ref, "bf16", 64, "clamped")


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_attention_strides_and_alignment(dev, kind):
    """Slices of one projection, heads first in memory, an odd offset (copied by the wrapper), a strided out, a broadcast key head."""
    n, H, G, D = [90, 33], 4, 2, 64
    sq = _starts(n)
    T = int(sq[-1])
    base = _randn((T, H + 2 * G, D), 1, kind)
    ref = opacked.attention(base[:, :H], base[:, H:H + G], base[:, H + G:], sq, sq, True)
    db, ds = base.to(dev), sq.to(dev)
    _check_attention(acnative.attention_packed(db[:, :H], db[:, H:H + G], db[:, H + G:], ds, causal=True), None, ref, kind, D, "slices")
    first = db.transpose(0, 1).contiguous().transpose(0, 1)
    _check_attention(acnative.attention_packed(first[:, :H], first[:, H:H + G], first[:, H + G:], ds, causal=True), None, ref, kind, D, "heads first")
    odd = torch.empty(T, H + 2 * G, D + 3, dtype=KINDS[kind], device=dev)[..., 1:D + 1]
    odd.copy_(db)
    _check_attention(acnative.attention_packed(odd[:, :H], odd[:, H:H + G], odd[:, H + G:], ds, causal=True), None, ref, kind, D, "odd")
    wide = torch.full((T, 2 * H, D + 16), 9.0, dtype=KINDS[kind], device=dev)
    out = wide[:, H:, 8:D + 8]
    acnative.attention_packed(db[:, :H], db[:, H:H + G], db[:, H + G:], ds, causal=True, out=out)
    _check_attention(out, None, ref, kind, D, "strided out")
    assert (wide[:, :H] == 9.0).all() and (wide[..., :8] == 9.0).all() and (wide[..., D + 8:] == 9.0).all()
    one = base[:, H:H + 1].expand(T, G, D)
    ref1 = opacked.attention(base[:, :H], one, base[:, H + G:], sq, sq, False)
    _check_attention(acnative.attention_packed(db[:, :H], db[:, H:H + 1].expand(T, G, D), db[:, H + G:], ds), None, ref1, kind, D, "broadcast")


def test_attention_single_token_with_odd_strides(dev):
    """A tensor of one token or one head may carry any stride for that axis."""
    base = _randn((3, 5, 64), 1, "bf16").to(dev)
    q = base.as_strided((1, 5, 64), (321, 64, 1))
    out = torch.zeros(400, dtype=torch.bfloat16, device=dev).as_strided((1, 5, 64), (333, 64, 1))
    starts = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    acnative.attention_packed(q, q, q, starts, out=out)
    assert torch.equal(out, q)                                      # one key: its value
    one = base[:, :1].as_strided((3, 1, 64), (320, 7, 1))
    got = acnative.attention_packed(one, one, one, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev))
    assert torch.equal(got, one)


def test_attention_is_the_same_every_time(dev):
    sq, sk = _starts([1, 5, 260]), _starts([3000, 900, 1500])
    args = [t.to(dev) for t in (_randn((266, 8, 128), 1, "bf16"), _randn((5400, 2, 128), 2, "bf16"), _randn((5400, 2, 128), 3, "bf16"), sq, sk)]
    first = acnative.attention_packed(*args, causal=True, max_q=260, max_k=3000)
    for _ in range(3):
        assert torch.equal(first, acnative.attention_packed(*args, causal=True, max_q=260, max_k=3000))


def test_on_another_stream_and_in_graphs(dev):
    """Two graphs captured on one stream, replayed in turn with other inputs and eager work between: each equals the eager result."""
    H, G, D = 8, 2, 64
    sq, sk = _starts([1, 1, 1]).to(dev), _starts([2000, 3000, 10]).to(dev)
    freq, side = acnative.rotary_frequencies(D, device=dev), torch.cuda.Stream()

    def make(seed):
        q, k, v = _randn((3, H, D), seed, "bf16").to(dev), _randn((5010, G, D), seed + 1, "bf16").to(dev), _randn((5010, G, D), seed + 2, "bf16").to(dev)
        pos = torch.tensor([2000 + seed, 3000, 10], dtype=torch.int32, device=dev)

        def step():
            return acnative.attention_packed(acnative.rotary(q, None, pos, freq), k, v, sq, sk, max_q=1, max_k=3000, causal=True)
        return q, step

    made = [make(1), make(11)]
    eager = []
    with torch.cuda.stream(side):
        for _, step in made:
            eager.append(step())
    side.synchronize()
    graphs = []
    for _, step in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    for turn in range(3):
        for (g, _), (q, _) in zip(graphs, made):
            g.replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, eager):
            assert torch.equal(out, want)
        for i, (q, step) in enumerate(made):
            q.mul_(0.5)
            eager[i] = step()
        torch.cuda.synchronize()


def test_offsets_that_pass_32_bits(dev):
    """A key buffer of more than 2^32 bytes: the last sequence's keys lie behind them."""
    G, D, n = 8, 128, 2_100_000                                     # 2.1e6 tokens x 2 KB = 4.3 GB each
    k = torch.zeros(n, G, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros(n, G, D, dtype=torch.bfloat16, device=dev)
    tail = 300
    k[-tail:] = _randn((tail, G, D), 1, "bf16").to(dev)
    v[-tail:] = _randn((tail, G, D), 2, "bf16").to(dev)
    q = _randn((5, G, D), 3, "bf16")
    sq, sk = torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([0, n - tail, n], dtype=torch.int32)
    got = acnative.attention_packed(q.to(dev), k, v, sq.to(dev), sk.to(dev), max_q=3, max_k=n, causal=True)
    local = _starts([tail])
    ref = opacked.attention(q[2:], k[-tail:].cpu(), v[-tail:].cpu(), _starts([3]), local, True)
    _check_attention(got[2:], None, ref, "bf16", D, "far")
    assert (got[:2] == 0).all()                                     # all values of the first sequence are zero
    turned = acnative.rotary(k, None, torch.zeros(n, dtype=torch.int32, device=dev), acnative.rotary_frequencies(D, device=dev))
    assert torch.equal(turned[-tail:], k[-tail:])


def test_images_of_their_own_sizes_as_a_backbone_would(dev):
    """Rotary rows and columns, then attention, over a packed batch of patch grids: against the oracle's chain."""
    grids = [(4, 6), (28, 28), (1, 1), (9, 16)]
    H, D = 12, 64
    lengths = [1 + a * b for a, b in grids]
    pos = torch.cat([torch.cat([torch.zeros(2, 1, dtype=torch.int64), torch.stack([torch.arange(a * b) // b, torch.arange(a * b) % b])], 1) for a, b in grids], 1)
    starts, longest = acnative.sequence_starts(lengths, dev)
    assert longest == 785 and starts.cpu().tolist() == _starts(lengths).tolist()
    T = sum(lengths)
    qkv = _randn((T, 3 * H, D), 4, "fp32")
    freq = acnative.rotary_frequencies(D, 100.0, axes=2)
    d = qkv.to(dev)
    q, k = acnative.rotary(d[:, :H], d[:, H:2 * H], pos.to(dev), freq.to(dev))
    got, sums = acnative.attention_packed(q, k, d[:, 2 * H:], starts, max_q=longest, max_k=longest, want_sums=True)
    rq, _ = opacked.rotary(qkv[:, :H], pos, freq, "half", 0, 1.0)
    rk, _ = opacked.rotary(qkv[:, H:2 * H], pos, freq, "half", 0, 1.0)
    ref = opacked.attention(rq, rk, qkv[:, 2 * H:], starts.cpu(), starts.cpu(), False)
    ref["score"] = ref["score"] * (1 + 2.0 ** -20 / E / (2 * D + 6))          # the turned q and k are off by 2^-21 each
    _check_attention(got, sums, ref, "fp32", D, "chain")


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("lengths", [([200, 30], None), ([1, 2], [300, 700])])
def test_attention_with_infinite_keys_and_values(dev, kind, lengths):
    """What rows do see: a key whose scores are -inf is left out, one at +inf makes NaN, infinite values pass where they weigh."""
    queries, keys = lengths
    sq, sk = _starts(queries), _starts(keys or queries)
    H, D = 2, 64
    q = _randn((int(sq[-1]), H, D), 1, kind).abs() + 0.125                  # positive: the sign of an infinite key decides
    k, v = _randn((int(sk[-1]), H, D), 2, kind), _randn((int(sk[-1]), H, D), 3, kind)
    k[5, 0, 3] = -math.inf
    v[9, 1, 4] = math.inf
    v[10, 1, 5] = math.nan
    ref = opacked.attention(q, torch.where(torch.isinf(k), torch.zeros_like(k), k), v, sq, sk, False)
    # without key 5 for head 0 of the first sequence
    keep = torch.ones(int(sk[-1]), dtype=torch.bool)
    keep[5] = False
    lens = [n for n in (keys or queries)]
    lens[0] -= 1
    less = opacked.attention(q, k[keep], v[keep], sq, _starts(lens), False)
    first = slice(0, queries[0])
    for key in ref:
        ref[key][first, 0] = less[key][first, 0]
    args = [t.to(dev) for t in (q, k, v, sq, sk)]
    got, sums = acnative.attention_packed(*args, want_sums=True)
    _check_attention(got, sums, ref, kind, D, "infinite")
    k[7, 0, 1] = math.inf
    got = acnative.attention_packed(args[0], k.to(dev), *args[2:]).cpu()
    assert torch.isnan(got[first, 0]).all() and torch.equal(got[first, 1].isnan(), ref["out"][first, 1].isnan())
    assert torch.isfinite(got[queries[0]:]).all()
    k[:] = -math.inf                                                         # no score above -inf: zero
    got, sums = acnative.attention_packed(args[0], k.to(dev), torch.nan_to_num(v).to(dev), *args[3:], want_sums=True)
    assert (got == 0).all() and (sums == -math.inf).all()


def test_attention_large_and_small_magnitudes_in_fp32(dev):
    """fp32 in thirds: values near the largest float and far under 1 keep their digits."""
    sq = _starts([90, 40])
    for scale in (1e30, 1e-30):
        q, k, v = _randn((130, 2, 64), 1, "fp32"), _randn((130, 2, 64), 2, "fp32"), _randn((130, 2, 64), 3, "fp32") * scale
        ref = opacked.attention(q, k, v, sq, sq, True)
        got = acnative.attention_packed(q.to(dev), k.to(dev), v.to(dev), sq.to(dev), causal=True)
        err = (got.cpu().double() - ref["out"]).abs()
        assert (err <= _u("fp32") * ref["out"].abs() + (2 * (2 * 64 + 6) * E * ref["score"] + (ref["keys"] + 8) * E)[..., None] * ref["weighted"]).all()
        q2, k2 = q * 1e15, k * 1e-15
        got = acnative.attention_packed(q2.to(dev), k2.to(dev), q.to(dev), sq.to(dev), causal=True)
        ref2 = opacked.attention(q2, k2, q, sq, sq, True)
        err = (got.cpu().double() - ref2["out"]).abs()
        assert (err <= _u("fp32") * ref2["out"].abs() + (2 * (2 * 64 + 6) * E * ref2["score"] + (ref2["keys"] + 8) * E)[..., None] * ref2["weighted"]).all()


def test_attention_many_sequences(dev):
    """More than 64 sequences (not ordered by length), and a thousand short ones."""
    g = torch.Generator().manual_seed(4)
    for count, top in ((65, 200), (1000, 9)):
        n = torch.randint(0, top, (count,), generator=g).tolist()
        _run(dev, "bf16", 4, 2, 64, n, causal=True, seed=count)
        _run(dev, "fp16", 2, 2, 32, [1] * count, [x + 1 for x in n], causal=True, seed=count + 1)


def test_attention_both_calls_at_once(dev):
    """Two streams at a time, each with its own split key axis: the same as one after the other."""
    sq, sk = _starts([1, 1]).to(dev), _starts([6000, 5000]).to(dev)
    sets = [[_randn((2, 8, 128), i, "bf16").to(dev), _randn((11000, 2, 128), i + 1, "bf16").to(dev), _randn((11000, 2, 128), i + 2, "bf16").to(dev)] for i in (1, 11)]
    alone = [acnative.attention_packed(*s, sq, sk, max_q=1, max_k=6000, causal=True) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(acnative.attention_packed(*s, sq, sk, max_q=1, max_k=6000, causal=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_the_attention_half_of_a_block(dev, kind):
    """Norm, projection, rotary positions, attention over images of their own sizes; then the norm's gradients from the projection's:
    each step against float64 on the step's own input."""
    grids, H, G, D = [(3, 5), (12, 12), (1, 1), (7, 20)], 6, 2, 32
    C = H * D
    lengths = [a * b + 1 for a, b in grids]
    T = sum(lengths)
    pos = torch.cat([torch.cat([torch.zeros(2, 1, dtype=torch.int64), torch.stack([torch.arange(a * b) // b, torch.arange(a * b) % b])], 1) for a, b in grids], 1)
    starts, longest = acnative.sequence_starts(lengths, dev)
    x, dy = _randn((T, C), 1, kind).to(dev), _randn((T, C), 2, kind).to(dev)
    w, b = (1 + 0.2 * _randn((C,), 3, "fp32")).to(dev), _randn((C,), 4, "fp32").to(dev)
    proj = (_randn(((H + 2 * G) * D, C), 5, "fp32") / C ** 0.5).to(KINDS[kind]).to(dev)
    freq = acnative.rotary_frequencies(D, 100.0, axes=2, device=dev)
    y, mean, rstd = acnative.layer_norm(x, w, b, want_stats=True)
    xd = x.cpu().double().requires_grad_()
    wd = w.cpu().double().requires_grad_()
    bd = b.cpu().double().requires_grad_()
    yd = torch.nn.functional.layer_norm(xd, (C,), wd, bd, 1e-6)
    assert ((y.cpu().double() - yd).abs() <= _u(kind) * yd.abs() + 1e-5).all()
    qkv = (y.float() @ proj.float().T).to(KINDS[kind]).view(T, H + 2 * G, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    rq, sq_ = opacked.rotary(q.cpu(), pos, freq.cpu(), "half", 0, 1.0)
    acnative.rotary(q, k, pos.to(dev), freq, out_q=q, out_k=k)
    assert ((q.cpu().double() - rq).abs() <= _u(kind) * rq.abs() + (2.0 ** -22 + 4 * E) * sq_).all()
    got, sums = acnative.attention_packed(q, k, v, starts, max_q=longest, max_k=longest, want_sums=True)
    ref = opacked.attention(q.cpu(), k.cpu(), v.cpu(), starts.cpu(), starts.cpu(), False)
    _check_attention(got, sums, ref, kind, D, "half block")
    dx, dw, db = acnative.layer_norm_backward(dy, x, w, mean, rstd)
    gx, gw, gb = torch.autograd.grad(yd, (xd, wd, bd), dy.cpu().double())
    assert ((dx.cpu().double() - gx).abs() <= _u(kind) * gx.abs() + 2e-5 * gx.abs().max()).all()
    assert ((dw.cpu().double() - gw).abs() <= 1e-5 * (1 + gw.abs().max())).all() and ((db.cpu().double() - gb).abs() <= 1e-5 * (1 + gb.abs().max())).all()


def test_wrappers_refuse_what_they_say(dev):
    x = torch.zeros(8, 4, 64, device=dev)
    starts = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    freq = acnative.rotary_frequencies(64, device=dev)
    pos = torch.zeros(8, dtype=torch.int32, device=dev)
    a = acnative.attention_packed
    for error, call in (
            (TypeError, lambda: a(x, x.half(), x, starts)), (TypeError, lambda: a(x.double(), x.double(), x.double(), starts)),
            (ValueError, lambda: a(x, x[:, :, :32], x[:, :, :32], starts)), (ValueError, lambda: a(x, x[:, :2], x, starts)),
            (RuntimeError, lambda: a(x, x[:, :3], x[:, :3], starts)), (TypeError, lambda: a(x, x, x, starts.long())),
            (RuntimeError, lambda: a(x, x, x, starts.cpu())), (ValueError, lambda: a(x, x[:4], x[:4], starts)),
            (ValueError, lambda: a(x, x, x, starts, starts[:1])), (ValueError, lambda: a(x[0], x[0], x[0], starts)),
            (ValueError, lambda: a(x, x, x, starts, out=x)), (ValueError, lambda: a(x, x, x, starts, out=x.new_zeros(8, 4, 32).repeat(1, 1, 2)[:, :2])),
            (ValueError, lambda: a(x, x, x, starts, out=x.new_zeros(8, 1, 64).expand(8, 4, 64))), (RuntimeError, lambda: a(x, x, x, starts, scale=math.inf)),
            (ValueError, lambda: a(x.transpose(1, 2), x.transpose(1, 2), x.transpose(1, 2), starts)),
            (RuntimeError, lambda: a(x.clone().requires_grad_(), x, x, starts)),
            (ValueError, lambda: acnative.rotary(x, None, pos, freq, layout="other")), (TypeError, lambda: acnative.rotary(x, None, pos.float(), freq)),
            (TypeError, lambda: acnative.rotary(x, None, pos, freq.float())), (ValueError, lambda: acnative.rotary(x, None, pos[:4], freq)),
            (RuntimeError, lambda: acnative.rotary(x, None, pos, freq, offset=2)), (ValueError, lambda: acnative.rotary(x, x[:4], pos, freq)),
            (ValueError, lambda: acnative.rotary(x, None, pos, freq, out_k=x)), (ValueError, lambda: acnative.rotary(x[:, :2], x[:, 2:], pos, freq, out_q=x[:, 1:3])),
            (ValueError, lambda: acnative.layer_norm(x, torch.ones(32, device=dev))), (TypeError, lambda: acnative.layer_norm(x, torch.ones(64, device=dev).half())),
            (ValueError, lambda: acnative.layer_norm(x[:4], out=x[1:5])), (RuntimeError, lambda: acnative.layer_norm(x.clone().requires_grad_())),
            (ValueError, lambda: acnative.layer_norm_backward(x[:2], x, None, x[:, :, 0].contiguous(), x[:, :, 0].contiguous())),
            (ValueError, lambda: acnative.layer_norm_backward(x, x, None, pos.float(), pos.float()))):
        with pytest.raises(error):
            call()
    assert acnative.attention_packed(x, x, x, starts, max_q=10 ** 12, max_k=10 ** 12).shape == x.shape


def test_rotary_more_tokens_than_one_launch_takes(dev):
    n = (16 << 20) + 37                                             # 16 tokens to a block, 2^20 blocks to a launch
    gen = torch.Generator(device=dev).manual_seed(5)
    q = torch.randn((n, 1, 2), generator=gen, device=dev).bfloat16()
    p = torch.randint(0, 4000, (n,), generator=gen, device=dev, dtype=torch.int32)
    f = torch.tensor([0.37], dtype=torch.float64, device=dev)
    got = acnative.rotary(q, None, p, f)
    got = got[0] if isinstance(got, tuple) else got
    for a, b in ((0, 100), ((16 << 20) - 60, n)):
        part = acnative.rotary(q[a:b], None, p[a:b].contiguous(), f)
        assert torch.equal(got[a:b], part[0] if isinstance(part, tuple) else part)


def test_attention_many_sequences_without_bounds(dev):
    """The bound of every sequence is then the number of tokens: more blocks than a launch has, so they walk over the tiles."""
    lengths = [50000] + [(37 * i) % 131 for i in range(2000)]
    starts = _starts(lengths).to(dev)
    T = sum(lengths)
    gen = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn((T, 36, 64), generator=gen, device=dev).bfloat16()
    q, k, v = qkv[:, :12], qkv[:, 12:24], qkv[:, 24:]
    got = acnative.attention_packed(q, k, v, starts)
    # the same tiles and keys in the same order: the same bits
    n = 50000
    one = acnative.attention_packed(q[:n], k[:n], v[:n], torch.tensor([0, n], dtype=torch.int32, device=dev))
    assert torch.equal(got[:n], one)
    rest = acnative.attention_packed(q[n:], k[n:], v[n:], starts[1:] - n, max_q=130, max_k=130)
    assert torch.equal(got[n:], rest)
