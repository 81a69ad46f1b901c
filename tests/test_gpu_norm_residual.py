"""h3hip_norm_modulate and h3hip_gated_residual on the GPU against their formulas in 64 bits.

What is rounded to fp32 (u = 2^-24 each, relative). A row's mean square: a square (1) and its
sum, a thread's 16 terms, 6 steps of a wave and 3 + 2 of the waves (27 at most), the width's
inverse and its product (2), eps (1): 31 u, halved by the inverse root, whose own error is 2 u:
the normalised value, a product, is off by less than 19 u. Times gamma (1 + scale), itself
3 u: 23 u of N = |v rs gamma (1 + scale)|; the shift's sum adds u of both: h is off by 24 u N +
u |shift|, and by its store's 2^-8 |h|. r = a x + gate z: a product u |a x|, z's 19 u, the
product of the tables u, theirs u, the sum u of both: less than 24 u (|a x| + |gate z|), and the
store's 2^-8 |r|. h of a next norm takes the fp32 r: d = 24 u (|a x| + |gate z|) of each
element, and of the row's root mean square at most the largest d's share, so N's error grows by
(d + |r| max(d) / rms) rs |gamma (1 + scale)|. bf16 subnormals are off by 2^-134."""
import pytest
import torch

from _gpu import note
from _mx4 import bits16

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
SIZES = [(1, 1), (1, 5376), (3, 7), (5, 33), (7, 64), (2, 511), (9, 512), (4, 513), (65, 1000),
         (300, 1001), (33, 2048), (17, 2051), (125, 5120), (3000, 640), (1151, 5376), (40, 7168),
         (21, 8191), (6, 8192), (5, 8193), (12, 9000), (3, 16383), (4, 16384), (700, 3)]


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _inputs(S, H, seed, segments=1, special=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rows():
        t = (_randn(g, S, H) * torch.exp(2 * _randn(g, S, 1))).to(torch.bfloat16)
        if special and S > 4:
            t[2] = 0.0
            t[3] = (t[3].float() * 1e-30).to(torch.bfloat16)
            t[4] = (t[4].float() * 1e12).to(torch.bfloat16)
        return t
    tab = {k: (0.5 * _randn(g, segments, H)).to(torch.bfloat16) for k in ("scale", "shift", "gate")}
    tab["gamma"], tab["post"] = ((1 + 0.2 * _randn(g, H)).to(torch.bfloat16) for _ in range(2))
    return rows(), rows(), tab


def _segment(S, starts):
    r = torch.arange(S, device="cuda")
    return sum((r >= s).long() for s in starts[1:]) if len(starts) > 1 else torch.zeros_like(r)


def _norm64(v, d, tab, seg):
    """h of float64 rows v known to within d, and its bound."""
    ms = v.square().mean(1, keepdim=True)
    rs = 1 / torch.sqrt(ms + EPS)
    one = torch.ones((), dtype=torch.float64, device="cuda")
    f = tab["gamma"].double() if tab.get("gamma") is not None else one
    if tab.get("scale") is not None:
        f = f * (1 + tab["scale"].double()[seg])
    f = f.expand_as(v) if f.dim() < 2 else f
    shift = tab["shift"].double()[seg] if tab.get("shift") is not None else torch.zeros_like(v)
    h = v * rs * f + shift
    drift = (d + v.abs() * d.amax(1, keepdim=True) * rs) * rs * f.abs()
    return h, 24 * U * (v * rs * f).abs() + U * shift.abs() + drift + 2.0 ** -8 * h.abs() + 2.0 ** -133


def _after64(x, y, tab, alpha, post, seg):
    z = y.double()
    if post:
        z = z / torch.sqrt(z.square().mean(1, keepdim=True) + EPS) * tab["post"].double()
    if tab.get("gate") is not None:
        z = z * tab["gate"].double()[seg]
    a = alpha * x.double()
    return a + z, 24 * U * (a.abs() + z.abs())


def _check(name, got, want, bound):
    d = (got.double() - want).abs()
    worst = float((d / bound).max()) if d.numel() else 0.0
    print(f"{name}: worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0, name


def _run_before(S, H, seed, starts=None, **drop):
    from h3hip import ops
    n = len(starts) if starts else 1
    x, _, tab = _inputs(S, H, seed, n)
    t = {k: None if drop.get(k) else tab[k] for k in ("gamma", "scale", "shift")}
    note(f"norm_modulate S={S} H={H} starts={starts} without={sorted(drop)}")
    h = ops.norm_modulate(x, **t, segments=starts, eps=EPS)
    torch.cuda.synchronize()
    want, bound = _norm64(x.double(), torch.zeros_like(x, dtype=torch.float64), t,
                          _segment(S, starts or [0]))
    _check("h", h, want, bound)


@pytest.mark.parametrize("S,H", SIZES)
def test_before_against_64_bits(h3, S, H):
    _run_before(S, H, S + H)


@pytest.mark.parametrize("S,H", SIZES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("chained", [False, True])
def test_after_against_64_bits(h3, S, H, post, chained):
    from h3hip import ops
    x, y, tab = _inputs(S, H, S + H + 1)
    alpha = 0.875 if post else 1.0
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}
    note(f"gated_residual S={S} H={H} post={post} chained={chained}")
    got = ops.gated_residual(x, y, tab["gate"], post_gamma=tab["post"] if post else None,
                             residual_scale=alpha, eps=EPS, next_norm=norm if chained else None)
    torch.cuda.synchronize()
    seg = _segment(S, [0])
    r, d = _after64(x, y, tab, alpha, post, seg)
    if not chained:
        got = (got,)
    _check("r", got[0], r, d + 2.0 ** -8 * r.abs() + 2.0 ** -133)
    if chained:
        _check("h", got[1], *_norm64(r, d, norm, seg))
        alone = ops.gated_residual(x, y, tab["gate"], post_gamma=tab["post"] if post else None,
                                   residual_scale=alpha, eps=EPS)
        assert (bits16(alone) == bits16(got[0])).all()


@pytest.mark.parametrize("starts", [[0], [0, 1], [0, 5, 5, 9], [0, 0, 0], [0, 100], [0, 17, 40],
                                    [0, 40, 40], list(range(16)), [0, 39]])
@pytest.mark.parametrize("S,H", [(1, 100), (40, 1000), (40, 9000)])
def test_segments(h3, S, H, starts):
    """Of no rows, past the end, of one row: each row takes its own segment's tables."""
    from h3hip import ops
    _run_before(S, H, 3, starts)
    x, y, tab = _inputs(S, H, 5, len(starts))
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}
    r, h = ops.gated_residual(x, y, tab["gate"], segments=starts, eps=EPS, next_norm=norm)
    seg = _segment(S, starts)
    want, d = _after64(x, y, tab, 1.0, False, seg)
    _check("r", r, want, d + 2.0 ** -8 * want.abs() + 2.0 ** -133)
    _check("h", h, *_norm64(want, d, norm, seg))


@pytest.mark.parametrize("missing", [("gamma",), ("scale",), ("shift",), ("gamma", "scale", "shift"),
                                     ("scale", "shift")])
def test_optional_tables(h3, missing):
    from h3hip import ops
    _run_before(50, 1000, 7, [0, 20], **{k: True for k in missing})
    x, y, tab = _inputs(50, 1000, 8, 2)
    norm = {k: tab[k] for k in ("gamma", "scale", "shift") if k not in missing}
    r, h = ops.gated_residual(x, y, segments=[0, 20], eps=EPS, next_norm=norm, post_gamma=tab["post"])
    seg = _segment(50, [0, 20])
    want, d = _after64(x, y, {"post": tab["post"]}, 1.0, True, seg)
    _check("r", r, want, d + 2.0 ** -8 * want.abs() + 2.0 ** -133)
    _check("h", h, *_norm64(want, d, norm, seg))


def test_one_segment_tables_as_vectors(h3):
    from h3hip import ops
    x, y, tab = _inputs(30, 777, 1)
    flat = {k: tab[k].reshape(-1) for k in ("scale", "shift", "gamma")}
    a = ops.norm_modulate(x, tab["gamma"], tab["scale"], tab["shift"])
    b = ops.norm_modulate(x, **flat)
    assert (bits16(a) == bits16(b)).all()
    assert (bits16(ops.gated_residual(x, y, tab["gate"])) ==
            bits16(ops.gated_residual(x, y, tab["gate"][0]))).all()


@pytest.mark.parametrize("S,H,first", [(20, 1000, 0), (20, 1001, 3), (7, 33, 1), (5, 9001, 5)])
def test_strides_addresses_and_what_is_not_written(h3, S, H, first):
    """Every tensor at an address and with strides of its own."""
    from h3hip import ops
    x, y, tab = _inputs(S, H, 9, 3)
    starts = [0, 2, S - 1]

    def wide(t, gap):
        ld = t.shape[1] + gap
        buf = torch.full((t.shape[0] * ld + first,), 7.0, dtype=torch.bfloat16, device="cuda")
        v = buf[first:].view(t.shape[0], ld)[:, :t.shape[1]]
        v.copy_(t)
        return buf, v
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}
    want = ops.gated_residual(x, y, tab["gate"], post_gamma=tab["post"], segments=starts,
                              next_norm=norm)
    one = wide(tab["gamma"][None], 0)[1][0]
    far = dict(gamma=one, scale=wide(tab["scale"], 5)[1], shift=wide(tab["shift"], 9)[1])
    rbuf, r = wide(torch.zeros_like(x), 3)
    hbuf, h = wide(torch.zeros_like(x), 11)
    note(f"gated_residual strided S={S} H={H} first={first}")
    got = ops.gated_residual(wide(x, 1)[1], wide(y, 6)[1], wide(tab["gate"], 2)[1],
                             post_gamma=wide(tab["post"][None], 0)[1][0], segments=starts,
                             next_norm=far, out=(r, h))
    assert got[0] is r and got[1] is h
    for buf, v, ref in ((rbuf, r, want[0]), (hbuf, h, want[1])):
        assert (bits16(v) == bits16(ref)).all()
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[first:].view(S, -1)[:, :H] = False
        assert (buf[rest] == 7.0).all()
    hb, hv = wide(torch.zeros_like(x), 4)
    ops.norm_modulate(wide(x, 1)[1], **far, segments=starts, out=hv)
    assert (bits16(hv) == bits16(ops.norm_modulate(x, **norm, segments=starts))).all()


@pytest.mark.parametrize("S,H", [(1, 100), (3000, 1000), (2000, 5120), (50, 10000)])
def test_in_place(h3, S, H):
    """The residual stream, or the block's output, overwritten by r or h."""
    from h3hip import ops
    x, y, tab = _inputs(S, H, 4)
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}
    want = ops.gated_residual(x, y, tab["gate"], post_gamma=tab["post"], next_norm=norm)
    note(f"norms in place S={S} H={H}")
    for ri, hi in ((0, None), (1, None), (0, 1), (1, 0), (None, 0)):
        ins = [x.clone(), y.clone()]
        r = ins[ri] if ri is not None else torch.empty_like(x)
        h = ins[hi] if hi is not None else torch.empty_like(x)
        ops.gated_residual(*ins, tab["gate"], post_gamma=tab["post"], next_norm=norm, out=(r, h))
        assert (bits16(r) == bits16(want[0])).all() and (bits16(h) == bits16(want[1])).all()
    h = ops.norm_modulate(x, **norm)
    c = x.clone()
    assert (bits16(ops.norm_modulate(c, **norm, out=c)) == bits16(h)).all()


def test_rows_that_are_not_finite(h3):
    """An infinity or a NaN stays in its row."""
    from h3hip import ops
    x, y, tab = _inputs(40, 1000, 6, special=False)
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}
    clean = ops.gated_residual(x, y, tab["gate"], post_gamma=tab["post"], next_norm=norm)
    x2, y2 = x.clone(), y.clone()
    x2[3, 5], y2[9, 999] = float("nan"), float("inf")
    got = ops.gated_residual(x2, y2, tab["gate"], post_gamma=tab["post"], next_norm=norm)
    keep = [i for i in range(40) if i not in (3, 9)]
    for a, b in zip(got, clean):
        assert (bits16(a[keep]) == bits16(b[keep])).all()
    assert torch.isnan(got[0][3, 5]) and torch.isnan(got[0][9, 999])
    assert torch.isnan(got[1][3]).all() and torch.isnan(got[1][9]).all()


@pytest.mark.parametrize("H", [100, 1000, 5120, 9000])
def test_rows_do_not_depend_on_the_others(h3, H):
    from h3hip import ops
    x, y, tab = _inputs(3000, H, 2)
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}

    def run(n):
        return ops.gated_residual(x[:n], y[:n], tab["gate"], post_gamma=tab["post"], next_norm=norm)
    every = run(3000)
    for n in (1, 17, 1100):
        for a, b in zip(run(n), every):
            assert (bits16(a) == bits16(b[:n])).all()


def test_no_rows(h3):
    from h3hip import ops
    x = torch.empty((0, 50), dtype=torch.bfloat16, device="cuda")
    assert ops.norm_modulate(x).shape == (0, 50)
    assert [t.shape for t in ops.gated_residual(x, x, next_norm={})] == [(0, 50)] * 2


def test_too_wide_is_declined(h3):
    from h3hip import ops
    x = torch.zeros((2, 16385), dtype=torch.bfloat16, device="cuda")
    assert ops.norm_modulate(x) is None and ops.gated_residual(x, x) is None


def test_offsets_past_32_bits(h3):
    from h3hip import ops
    S, H = 500_000, 4608
    x = torch.zeros((S, H), dtype=torch.bfloat16, device="cuda")
    tail, _, tab = _inputs(20, H, 1)
    x[-20:] = tail
    note("norm_modulate large")
    h = ops.norm_modulate(x, tab["gamma"], tab["scale"], tab["shift"])
    want = ops.norm_modulate(tail, tab["gamma"], tab["scale"], tab["shift"])
    assert (bits16(h[-20:]) == bits16(want)).all()
    assert (bits16(h[:3]) == bits16(tab["shift"].expand(3, H))).all()


def test_captured_replayed_and_on_two_streams(h3):
    from h3hip import ops
    x, y, tab = _inputs(700, 1000, 1, 2)
    norm = {k: tab[k] for k in ("gamma", "scale", "shift")}

    def run(a, b):
        h = ops.norm_modulate(a, **norm, segments=[0, 100])
        return (h, *ops.gated_residual(a, b, tab["gate"], post_gamma=tab["post"],
                                       segments=[0, 100], next_norm=norm))
    run(x, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    note("norms captured")
    with torch.cuda.graph(graph):
        got = run(x, y)
    for rep in range(4):
        x.copy_(_inputs(700, 1000, rep + 5)[0])
        want = [bits16(t) for t in run(x, y)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all((bits16(a) == b).all() for a, b in zip(got, want)), rep
    sides = [(*_inputs(700, 1000, s)[:2], torch.cuda.Stream()) for s in (1, 2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(4):
        for i, (a, b, st) in enumerate(sides):
            with torch.cuda.stream(st):
                outs[i].append(run(a, b))
    torch.cuda.synchronize()
    for i, (a, b, _) in enumerate(sides):
        want = [bits16(t) for t in run(a, b)]
        for o in outs[i]:
            assert all((bits16(t) == w).all() for t, w in zip(o, want))


def test_one_modulation_for_every_segment(h3):
    """Tables expanded over the segments: a row stride of 0."""
    from h3hip import ops
    x, y, tab = _inputs(60, 1000, 3)
    wide = {k: tab[k].expand(4, 1000) for k in ("scale", "shift", "gate")}
    norm = dict(gamma=tab["gamma"], scale=wide["scale"], shift=wide["shift"])
    a = ops.gated_residual(x, y, wide["gate"], segments=[0, 5, 9, 30], next_norm=norm)
    b = ops.gated_residual(x, y, tab["gate"], next_norm=dict(gamma=tab["gamma"], scale=tab["scale"],
                                                             shift=tab["shift"]))
    for t, u in zip(a, b):
        assert (bits16(t) == bits16(u)).all()
    a = ops.norm_modulate(x, **norm, segments=[0, 5, 9, 30])
    assert (bits16(a) == bits16(ops.norm_modulate(x, tab["gamma"], tab["scale"], tab["shift"]))).all()
