"""The norms around the block (norm_modulate, norm_residual) and their backward against 64-bit arithmetic: types, widths from
one vector to the widest, equal and ragged samples, empty ones, padding rows that hold NaN, slots routed nowhere, row strides,
no rows.

Tolerances.  A row sum of d terms is taken by 64 or more lanes in turn (d / 64 terms at most in each), six exchange steps and
at most 16 waves: relative to the sum of the absolute terms it is off by at most row = (d / 64 + 24) 2^-24; the few further
fp32 steps of an element add less than 16 2^-24.  Then one rounding to the output's type.  A column sum over T rows goes
through at most T / 512 + 1 rows of a wave, 8 row groups, and T / 8 / 16 chunk sums + 16."""
import pytest
import torch

from tests import block_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _row_tol(d):
    return (d / 64 + 24 + 16) * R.EPS24


def _col_tol(T, d):
    return (T / 512 + 1 + 8 + T / 128 + 16) * R.EPS24 + _row_tol(d)


def _close(name, got, ref, slack):
    """|got - ref| <= slack (an fp32 bound per element) plus one rounding to got's type."""
    got64 = got.detach().cpu().double()
    assert got64.shape == ref.shape, (name, got64.shape, ref.shape)
    bound = slack + R.half_step(got.dtype) * (ref.abs() + slack) + R.tiny(got.dtype)
    bad = ~((got64 - ref).abs() <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((got64 - ref).abs() / bound).nan_to_num(nan=9e9).max()):.3g} of the bound")


def _starts(T, B, g, first=0, last=None):
    last = T if last is None else last
    cuts = torch.randint(first, last + 1, (B - 1,), generator=g).sort().values
    if B > 2:
        cuts[1] = cuts[0]  # an empty sample
    return [first] + cuts.tolist() + [last]


class _Case:
    def __init__(self, T, d, B, ragged, stream, block, weight, mods, seed=0, pad=(0, 0)):
        g = torch.Generator().manual_seed(seed + T + d)
        self.T, self.d, self.B, self.eps = T, d, B, EPS
        r = lambda *s, std=1.0, dt=FP: (torch.randn(*s, generator=g) * std).to(dt)
        self.starts = _starts(T, B, g, pad[0], T - pad[1]) if ragged else None
        self.b = R.sample_rows(T, B, self.starts)
        self.x = r(T, d, std=2.0, dt=stream)
        self.w = None if weight is None else (r(d, std=0.1) + 1).to(weight)
        self.scale, self.shift = (None, None) if mods is None else (r(B, d, std=0.3, dt=mods), r(B, d, std=0.5, dt=mods))
        self.gate = None if mods is None else r(B, d, std=0.4, dt=mods)
        self.dh, self.dres = r(T, d, std=0.3, dt=block), r(T, d, std=0.3, dt=stream)
        self.g, self.r = g, r
        # padding rows may hold anything
        off = self.b < 0
        self.x_bad = self.x.clone()
        self.x_bad[off] = float("nan")
        self.dh_bad = self.dh.clone()
        self.dh_bad[off] = float("nan")

    def dev(self, t):
        return None if t is None else t.cuda()

    def starts_dev(self):
        return None if self.starts is None else torch.tensor(self.starts, dtype=torch.int32, device="cuda")


CASES = [
    # T, d, B, ragged, stream, block, weight, mods, padding rows before / behind
    (1, 8, 1, False, BF, BF, BF, None, (0, 0)),
    (3, 64, 1, False, HF, HF, None, HF, (0, 0)),
    (7, 520, 7, False, FP, BF, FP, FP, (0, 0)),          # a sample per row
    (64, 1536, 4, False, BF, BF, BF, BF, (0, 0)),
    (300, 1000, 5, True, FP, HF, BF, FP, (3, 11)),
    (33, 2048, 40, True, FP, FP, FP, BF, (1, 2)),        # more samples than rows: most of them empty
    (1200, 1536, 3, True, BF, BF, None, FP, (0, 30)),
    (1029, 256, 1, False, BF, BF, FP, None, (0, 0)),
    (21, 2056, 3, False, BF, BF, FP, BF, (0, 0)),        # four waves per row
    (40, 5000, 2, True, HF, HF, HF, FP, (0, 1)),
    (19, 8192, 1, True, FP, BF, FP, FP, (2, 3)),
    (9, 8200, 3, False, BF, BF, BF, BF, (0, 0)),         # sixteen
    (6, 16384, 2, True, FP, HF, FP, FP, (1, 1)),
    (5000, 64, 611, True, BF, BF, BF, BF, (0, 9)),       # many samples inside one chunk of rows
    (2048, 136, 2048, False, BF, BF, BF, FP, (0, 0)),
    # equal samples of few rows, finished by the row groups themselves: a part of a workgroup's samples, one row each
    (20, 1536, 20, False, BF, BF, BF, BF, (0, 0)), (4500, 200, 1500, False, FP, BF, FP, FP, (0, 0)),
    (66, 4096, 33, False, HF, HF, HF, FP, (0, 0)), (5, 9000, 5, False, BF, BF, FP, BF, (0, 0)),
]
ids = [f"{c[0]}x{c[1]}_{c[2]}{'r' if c[3] else ''}" for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_norm_modulate(case):
    from trenowanie_generatora_obrazkow_amd import ops
    *a, pad = case
    c = _Case(*a, pad=pad)
    block = case[5]
    print("norm_modulate", case, flush=True)
    h = ops.norm_modulate(c.dev(c.x_bad), c.dev(c.w), c.dev(c.scale), c.dev(c.shift), c.starts_dev(), EPS, dtype=block)
    lv = [None if t is None else t.double().requires_grad_(True) for t in (c.x, c.w, c.scale, c.shift)]
    ref = R.norm_modulate(*lv, c.b, EPS)
    tol = _row_tol(c.d)
    with torch.no_grad():
        shift0 = 0 if c.shift is None else torch.where((c.b >= 0).unsqueeze(1), c.shift.double()[c.b.clamp(min=0)], 0.0)
        mag = (ref - shift0).abs() + (0 if c.shift is None else shift0.abs())
    _close("h", h, ref.detach(), tol * mag)
    assert (h[(c.b < 0).cuda()] == 0).all()

    # backward: u = dh, the gradient past the block joined with factor 0.5
    dx, dw, dsc, dsh = ops.norm_modulate_bwd(c.dev(c.dh_bad), c.dev(c.x_bad), c.dev(c.w), c.dev(c.scale), c.dev(c.shift),
                                             c.starts_dev(), EPS, dres=c.dev(c.dres), dres_scale=0.5)
    grads = torch.autograd.grad((ref * c.dh.double()).sum(), [t for t in lv if t is not None], allow_unused=True)
    it = iter(grads)
    rx, rw, rsc, rsh = (None if t is None else next(it) for t in lv)
    with torch.no_grad():
        live = (c.b >= 0).unsqueeze(1)
        x, u = torch.where(live, lv[0], 0.0), torch.where(live, c.dh.double(), 0.0)
        rr = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
        m = torch.ones(c.T, c.d, dtype=torch.float64)
        sc = m if c.scale is None else 1 + c.scale.double()[c.b.clamp(min=0)]
        w = m if c.w is None else c.w.double().expand_as(m)
        g = u * sc * w
        mag = (rr * g).abs() + x.abs() * rr ** 3 * (g * x).abs().mean(1, keepdim=True)
        _close("dx", dx, rx + 0.5 * c.dres.double(), 4 * tol * mag + 2 * R.EPS24 * c.dres.double().abs())
        n = x * rr
        ct = _col_tol(c.T, c.d)
        per = lambda v: torch.stack([v[c.b == i].sum(0) for i in range(c.B)])
        if c.w is not None:
            _close("dweight", dw, rw, ct * (u * sc * n).abs().sum(0))
        if c.scale is not None:
            _close("dscale", dsc, rsc, ct * per((u * w * n).abs()))
            _close("dshift", dsh, rsh, ct * per(u.abs()))


@pytest.mark.parametrize("case", CASES, ids=ids)
@pytest.mark.parametrize("k,shared,norm", [(1, False, True), (2, False, True), (3, True, True), (8, True, False)])
def test_norm_residual(case, k, shared, norm):
    from trenowanie_generatora_obrazkow_amd import ops
    *a, pad = case
    c = _Case(*a, seed=k, pad=pad)
    T, d, block = c.T, c.d, case[5]
    print("norm_residual", case, k, shared, norm, flush=True)
    y = c.r(T * k, d, std=0.5, dt=block)
    add = c.r(T, d, std=0.5, dt=block) if shared else None
    inv = torch.arange(T * k, dtype=torch.int32)
    inv[torch.rand(T * k, generator=c.g) < 0.1] = -1
    y_bad = y.clone()
    y_bad[inv < 0] = float("nan")                                      # rows no GEMM wrote
    y_bad.view(T, k, d)[c.b < 0] = float("inf")                        # padding rows
    s64 = R.slot_sum(y.double(), T, k, inv, None if add is None else add.double()).requires_grad_(True)
    lv = [None if t is None else t.double().requires_grad_(True) for t in (c.gate, c.w)]
    ref = R.norm_residual(s64, c.x.double(), lv[0], lv[1], norm, c.b, EPS, 0.75)
    kw = dict(gate=c.dev(c.gate), weight=c.dev(c.w), norm=norm, starts=c.starts_dev(), eps=EPS, k=k, inv_pos=inv.cuda(),
              add=c.dev(add))
    out = ops.norm_residual(y_bad.cuda(), c.dev(c.x), alpha=0.75, **kw)
    tol = _row_tol(d)
    with torch.no_grad():
        live = (c.b >= 0).unsqueeze(1)
        sabs = R.slot_sum(y.double().abs(), T, k, inv, None if add is None else add.double().abs())
        s = torch.where(live, s64, 0.0)
        rr = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS) if norm else torch.ones(T, 1, dtype=torch.float64)
        one = torch.ones(T, d, dtype=torch.float64)
        w = one if c.w is None else c.w.double().expand_as(one)
        gt = one if c.gate is None else c.gate.double()[c.b.clamp(min=0)]
        # the slots' sum is off by (k + 1) 2^-24 of the sum of their absolute values
        es = (k + 1) * R.EPS24 * sabs
        en = rr * es + rr ** 3 * s.abs() * (s.abs() * es).mean(1, keepdim=True) + tol * (s * rr).abs()
        _close("out", out, ref.detach(), torch.where(live, en * (w * gt).abs(), 0.0) + 4 * R.EPS24 * (0.75 * c.x.double()).abs())

    dout = c.r(T, d, std=0.3, dt=case[4])
    dy, dg, dw = ops.norm_residual_bwd(dout.cuda(), y_bad.cuda(), **kw)
    leaves = [s64] + [t for t in lv if t is not None]
    it = iter(torch.autograd.grad((ref * dout.double()).sum(), leaves, allow_unused=True))
    rs = next(it)
    rg, rw = (None if t is None else next(it) for t in lv)
    with torch.no_grad():
        u = torch.where(live, dout.double(), 0.0)
        g = u * w * gt
        n = s * rr
        eg = rr * g.abs()
        if norm:
            # derivative of r g - s r^3 mean(g s) in s, times the error of s, and the rounding of its own sums
            p = (g * s).abs().mean(1, keepdim=True)
            rel = (s.abs() * es).mean(1, keepdim=True) * rr ** 2
            slack = 4 * tol * (eg + s.abs() * rr ** 3 * p) + 4 * rel * (eg + s.abs() * rr ** 3 * p) \
                + es * rr ** 3 * p + s.abs() * rr ** 3 * (g.abs() * es).mean(1, keepdim=True)
        else:
            slack = tol * eg
        _close("dy", dy, rs, slack)
        assert (dy[(c.b < 0).cuda()] == 0).all()
        ct = _col_tol(T, d)
        per = lambda v: torch.stack([v[c.b == i].sum(0) for i in range(c.B)])
        en = torch.where(live, en, 0.0)
        if c.gate is not None:
            _close("dgate", dg, rg, ct * per((u * w * n).abs()) + per((u * w).abs() * en))
        if c.w is not None:
            _close("dweight", dw, rw, ct * (u * gt * n).abs().sum(0) + ((u * gt).abs() * en).sum(0))


def test_row_strides_and_shared_parameters():
    """x as columns of a wider matrix, parameters given once as (d,), and no parameter at all."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(50, 1000, generator=g).bfloat16().cuda()
    x = wide[:, 64:64 + 520]
    sc = (torch.randn(520, generator=g) * 0.3).cuda()
    y = torch.randn(50, 520, generator=g).bfloat16().cuda()
    assert torch.equal(ops.norm_modulate(x, scale=sc), ops.norm_modulate(x.contiguous(), scale=sc[None]))
    assert torch.equal(ops.norm_residual(y, x, gate=sc), ops.norm_residual(y, x.contiguous(), gate=sc[None]))
    dh = torch.randn(50, 520, generator=g).bfloat16().cuda()
    a, b = ops.norm_modulate_bwd(dh, x, scale=sc), ops.norm_modulate_bwd(dh, x.contiguous(), scale=sc[None])
    assert torch.equal(a[0], b[0]) and a[2].shape == sc.shape and torch.equal(a[2], b[2][0])
    assert a[1] is None and a[3] is None
    # the residual alone: alpha x + y
    out = ops.norm_residual(y, x, norm=False)
    assert torch.equal(out, (x.float() + y.float()).bfloat16())


def test_no_rows():
    from trenowanie_generatora_obrazkow_amd import ops
    x = torch.empty(0, 64, device="cuda", dtype=BF)
    w, sc = torch.ones(64, device="cuda", dtype=BF), torch.ones(3, 64, device="cuda")
    assert ops.norm_modulate(x, w, sc, sc).shape == (0, 64)
    dx, dw, dsc, dsh = ops.norm_modulate_bwd(x, x, w, sc, sc)
    assert dx.shape == (0, 64) and not dw.any() and not dsc.any() and not dsh.any()
    assert ops.norm_residual(x, x, gate=sc, weight=w).shape == (0, 64)
    dy, dg, dw = ops.norm_residual_bwd(x, x, gate=sc, weight=w)
    assert dy.shape == (0, 64) and not dg.any() and not dw.any()


def test_rows_of_zeros_and_infinities():
    """A zero row norms to zero (eps), an infinite element makes its own row NaN and no other."""
    from trenowanie_generatora_obrazkow_amd import ops
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(1))
    x[1] = 0
    x[2, 7] = float("inf")
    h = ops.norm_modulate(x.cuda()).cpu()
    assert (h[1] == 0).all() and torch.isfinite(h[[0, 3]]).all() and torch.isnan(h[2, 7])
    out = ops.norm_residual(x.cuda(), x.cuda()).cpu()
    assert (out[1] == 0).all() and torch.isfinite(out[[0, 3]]).all()


def test_gradients_against_differences():
    """Central differences of the kernels' own fp32 forward along random directions.  With step t the difference quotient
    has a truncation error of t^2 / 6 of the third derivative and a rounding error of 2^-24 |loss terms| / t: at t = 2^-5
    and unit-sized inputs both stay below 2e-3 of the sum of the terms' absolute values."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(3)
    T, d, t = 24, 64, 2.0 ** -5
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    x, w, sc, sh, u, y = r(T, d), r(d), r(4, d), r(4, d), r(T, d), r(2 * T, d)
    dx, dw, dsc, dsh = ops.norm_modulate_bwd(u, x, w, sc, sh)
    dy, dg, dw2 = ops.norm_residual_bwd(u, y, gate=sc, weight=w, k=2)
    f_in = lambda **k: (ops.norm_modulate(**{**dict(x=x, weight=w, scale=sc, shift=sh), **k}).double() * u.double())
    f_out = lambda **k: (ops.norm_residual(**{**dict(y=y, x=x, gate=sc, weight=w, k=2), **k}).double() * u.double())
    for f, name, v, grad in ((f_in, "x", x, dx), (f_in, "weight", w, dw), (f_in, "scale", sc, dsc), (f_in, "shift", sh, dsh),
                             (f_out, "gate", sc, dg), (f_out, "weight", w, dw2),
                             (f_out, "y", y, dy.repeat_interleave(2, 0))):
        e = torch.sign(torch.randn(v.shape, generator=g)).cuda() / 8
        hi, lo = f(**{name: v + t * e}), f(**{name: v - t * e})
        diff = float((hi - lo).sum() / (2 * t))
        want = float((grad.double() * e.double()).sum())
        size = float((grad.double() * e.double()).abs().sum()) + float(hi.abs().sum()) * 1e-2
        assert abs(diff - want) <= 2e-3 * size, (name, diff, want, size)


def test_two_streams_and_replays():
    """The same calls on another stream and captured in a graph: the eager bits, replay after replay, with inputs that
    change in between."""
    from trenowanie_generatora_obrazkow_amd import ops
    from trenowanie_generatora_obrazkow_amd.graphs import StepGraph
    g = torch.Generator().manual_seed(9)
    T, d, B = 600, 520, 3
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
    x, w, sc, sh, y, u = r(T, d), r(d), r(B, d), r(B, d), r(2 * T, d), r(T, d)
    starts = torch.tensor([0, 200, 201, 590], dtype=torch.int32, device="cuda")

    def step():
        h = ops.norm_modulate(x, w, sc, sh, starts)
        out = ops.norm_residual(y, x, gate=sc, weight=w, starts=starts, k=2)
        return (h, out, *ops.norm_modulate_bwd(u, x, w, sc, sh, starts, dres=u),
                *ops.norm_residual_bwd(u, y, gate=sc, weight=w, starts=starts, k=2))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = StepGraph(step)
    for rep in range(3):
        if rep:
            x.copy_(r(T, d))
            y.copy_(r(2 * T, d))
        want = [t.clone() for t in step()]
        got = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
