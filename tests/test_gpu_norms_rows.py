"""The norms and their backward where a workgroup walks many rows: every count of waves per row, samples that begin and end inside
a workgroup's rows, several of them or parts of three in one, padding before, between a workgroup's rows and behind, against
64-bit arithmetic on the GPU.

What a size reaches.  Forward: T waves-per-row / 4096 rows (two at least from 8192 rows of one wave, 4096 of two, 2048 of four,
1024 of eight and 512 of sixteen) for each row group in turn.  Backward: about T / 256 rows for a workgroup of 8, 4, 2, 1 and 1
row groups, so more than one batch from 2049, 1025, 513, 257 and 257 rows.

Tolerances.  A row sum of d terms is taken by 64 or more lanes in turn, six exchange steps and at most 16 waves, and the further
fp32 steps of an element add less than 16: row = (d / 64 + 40) 2^-24 of the sum of the absolute terms.  A column sum: at most
T / 256 + 8 rows of a wave, 8 row groups, T / 256 + 8 pieces of a workgroup, 8 + 32 steps over the workgroups: (T / 128 + 64) 2^-24
more.  Then one rounding to the output's type."""
import pytest
import torch

from tests import block_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # T, d, samples (None: B equal ones), B, stream, block, parameters, slots
    (17000, 64, "ragged", 40, BF, BF, BF, 2),            # one wave a row, one vector a lane
    (9001, 256, "ragged", 23, FP, BF, FP, 5),
    (9000, 1032, "ragged", 300, FP, FP, FP, 1),          # three vectors; samples shorter than a workgroup's rows
    (9000, 1536, None, 9, BF, BF, BF, 2),
    (5003, 1600, "ragged", 17, HF, HF, HF, 3),           # two waves
    (9000, 2056, "ragged", 31, BF, BF, FP, 1),
    (9000, 2056, None, 6, FP, HF, FP, 2),
    (4500, 4096, "ragged", 19, BF, BF, BF, 2),           # four
    (4500, 4104, "ragged", 150, FP, BF, FP, 1),
    (2100, 8192, "ragged", 12, FP, BF, FP, 2),           # eight
    (2100, 8200, "ragged", 90, BF, BF, BF, 1),
    (2100, 8200, None, 7, HF, HF, FP, 4),
    (1101, 16384, "ragged", 9, BF, BF, BF, 2),           # sixteen
    (1101, 12296, "ragged", 100, FP, BF, FP, 1),
    (1100, 16000, None, 4, FP, FP, FP, 1),
    # equal samples of few rows, taken whole by the row groups, several in turn
    (6000, 2048, None, 3000, BF, BF, BF, 2),
    (3000, 4096, None, 1500, BF, BF, FP, 1),
    (2100, 8200, None, 1050, BF, BF, FP, 2),
    (1200, 16384, None, 600, BF, BF, BF, 2),
    (900, 12296, None, 900, FP, HF, FP, 1),
]
ids = [f"{c[0]}x{c[1]}_{c[3]}{'r' if c[2] else ''}" for c in CASES]


class _Case:
    def __init__(self, T, d, samples, B, stream, block, par, k):
        g = torch.Generator(device="cuda").manual_seed(T + d + B)
        r = lambda *s, std=1.0, dt=FP: (torch.randn(*s, generator=g, device="cuda") * std).to(dt)
        self.T, self.d, self.B, self.k = T, d, B, k
        self.starts = None
        if samples:
            # odd places, an empty sample, runs of short ones next to long ones
            cuts = (torch.rand(B - 1, generator=g, device="cuda").square() * (T - 60)).long().sort().values + 13
            cuts[1] = cuts[0]
            self.starts = torch.cat([torch.tensor([7], device="cuda"), cuts, torch.tensor([T - 29], device="cuda")]).int()
        st = None if self.starts is None else self.starts.tolist()
        assert st is None or st == sorted(st)
        self.b = R.sample_rows(T, B, st).cuda()
        self.live = (self.b >= 0).unsqueeze(1)
        self.x, self.dh, self.dres = r(T, d, std=2.0, dt=stream), r(T, d, std=0.3, dt=block), r(T, d, std=0.3, dt=stream)
        self.y, self.dout = r(T * k, d, std=0.5, dt=block), r(T, d, std=0.3, dt=stream)
        self.w = (r(d, std=0.1) + 1).to(par)
        self.scale, self.shift, self.gate = r(B, d, std=0.3, dt=par), r(B, d, std=0.5, dt=par), r(B, d, std=0.4, dt=par)

    def bad(self, t, value, k=1):
        """t with another value in the padding rows."""
        return torch.where(self.live.repeat_interleave(k, 0), t, torch.full((), value, dtype=t.dtype, device="cuda"))

    def per(self, v):
        z = torch.zeros(self.B, self.d, dtype=torch.float64, device="cuda")
        return z.index_add_(0, self.b.clamp(min=0), torch.where(self.live, v, 0.0))


def _close(name, got, ref, slack):
    got64 = got.detach().double()
    assert got64.shape == ref.shape, (name, got64.shape, ref.shape)
    bound = slack + R.half_step(got.dtype) * (ref.abs() + slack) + R.tiny(got.dtype)
    bad = ~((got64 - ref).abs() <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[0].tolist()}, worst "
                           f"{float(((got64 - ref).abs() / bound).nan_to_num(nan=9e9).max()):.3g} of the bound")


def _tols(c):
    row = (c.d / 64 + 40) * R.EPS24
    return row, row + (c.T / 128 + 64) * R.EPS24


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_norm_modulate(case):
    from trenowanie_generatora_obrazkow_amd import ops
    c = _Case(*case)
    print("norm_modulate", case, flush=True)
    row, col = _tols(c)
    nan = float("nan")
    x, dh = c.bad(c.x, nan), c.bad(c.dh, nan)
    h = ops.norm_modulate(x, c.w, c.scale, c.shift, c.starts, EPS, dtype=case[5])
    lv = [t.double().requires_grad_(True) for t in (c.x, c.w, c.scale, c.shift)]
    ref = R.norm_modulate(*lv, c.b, EPS)
    with torch.no_grad():
        sh = torch.where(c.live, c.shift.double()[c.b.clamp(min=0)], 0.0)
        _close("h", h, ref, row * ((ref - sh).abs() + sh.abs()))
    got = ops.norm_modulate_bwd(dh, x, c.w, c.scale, c.shift, c.starts, EPS, dres=c.dres, dres_scale=0.5)
    rx, rw, rsc, rsh = torch.autograd.grad((ref * c.dh.double()).sum(), lv)
    with torch.no_grad():
        v, u = torch.where(c.live, lv[0], 0.0), torch.where(c.live, c.dh.double(), 0.0)
        rr = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        sc, w = 1 + c.scale.double()[c.b.clamp(min=0)], c.w.double()
        g, n = u * sc * w, v * rr
        mag = (rr * g).abs() + n.abs() * rr * (g * n).abs().mean(1, keepdim=True)
        _close("dx", got[0], rx + 0.5 * c.dres.double(), 4 * row * mag + 2 * R.EPS24 * c.dres.double().abs())
        _close("dweight", got[1], rw, col * (u * sc * n).abs().sum(0))
        _close("dscale", got[2], rsc, col * c.per((u * w * n).abs()))
        _close("dshift", got[3], rsh, col * c.per(u.abs()))
    # each parameter gradient by itself: the same bits
    for i, name in enumerate(("weight", "scale", "shift")):
        one = ops.norm_modulate_bwd(dh, x, c.w, c.scale, c.shift, c.starts, EPS, dres=c.dres, dres_scale=0.5, want=(name,))
        assert torch.equal(one[0], got[0]) and torch.equal(one[1 + i], got[1 + i])
        assert all(one[1 + j] is None for j in range(3) if j != i)


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_norm_residual(case):
    from trenowanie_generatora_obrazkow_amd import ops
    c = _Case(*case)
    k = c.k
    print("norm_residual", case, flush=True)
    row, col = _tols(c)
    y = c.bad(c.y, float("inf"), k)
    s = R.slot_sum(c.y.double(), c.T, k, None, None).requires_grad_(True)
    lv = [t.double().requires_grad_(True) for t in (c.gate, c.w)]
    ref = R.norm_residual(s, c.x.double(), lv[0], lv[1], True, c.b, EPS, 0.75)
    kw = dict(gate=c.gate, weight=c.w, starts=c.starts, eps=EPS, k=k)
    out = ops.norm_residual(y, c.x, alpha=0.75, **kw)
    with torch.no_grad():
        es = (k + 1) * R.EPS24 * R.slot_sum(c.y.double().abs(), c.T, k, None, None)  # the slots' sum is off by that
        v = torch.where(c.live, s, 0.0)
        rr = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        n, w, gt = v * rr, c.w.double(), c.gate.double()[c.b.clamp(min=0)]
        en = torch.where(c.live, rr * es + rr * n.abs() * (n.abs() * es).mean(1, keepdim=True) + row * n.abs(), 0.0)
        _close("out", out, ref, en * (w * gt).abs() + 4 * R.EPS24 * (0.75 * c.x.double()).abs())
    dy, dg, dw = ops.norm_residual_bwd(c.bad(c.dout, float("nan")), y, **kw)
    rs, rg, rw = torch.autograd.grad((ref * c.dout.double()).sum(), [s] + lv)
    with torch.no_grad():
        u = torch.where(c.live, c.dout.double(), 0.0)
        g = u * w * gt
        p = (g * n).abs().mean(1, keepdim=True)
        mag = rr * g.abs() + n.abs() * rr * p
        # the derivative of r (g - n mean(g n)) by s, times the error of s
        rel = (n.abs() * es).mean(1, keepdim=True) * rr
        slack = 4 * (row + rel) * mag + es * rr * rr * p + n.abs() * rr * rr * (g.abs() * es).mean(1, keepdim=True)
        _close("dy", dy, rs, torch.where(c.live, slack, 0.0))
        _close("dgate", dg, rg, col * c.per((u * w * n).abs()) + c.per((u * w).abs() * en))
        _close("dweight", dw, rw, col * (u * gt * n).abs().sum(0) + ((u * gt).abs() * en).sum(0))
    for i, name in enumerate(("gate", "weight")):
        one = ops.norm_residual_bwd(c.bad(c.dout, float("nan")), y, **kw, want=(name,))
        assert torch.equal(one[0], dy) and torch.equal(one[1 + i], (dg, dw)[i]) and one[2 - i] is None


@pytest.mark.parametrize("d", [64, 2056, 8200, 16384])
def test_output_over_the_stream(d):
    """The C entry's output may be x itself."""
    from trenowanie_generatora_obrazkow_amd import _lib as L, ops
    g = torch.Generator(device="cuda").manual_seed(d)
    T = 1100
    x, y, gate = (torch.randn(n, d, generator=g, device="cuda") for n in (T, 2 * T, 5))
    want = ops.norm_residual(y, x, gate=gate, k=2, alpha=0.5)
    L.call("hmoe_norm_residual", y.data_ptr(), None, 2, None, L.DT_F32, x.data_ptr(), d, L.DT_F32, None, 0, gate.data_ptr(),
           L.DT_F32, None, 5, T, d, 1, EPS, 0.5, x.data_ptr(), L.stream(x.device))
    assert torch.equal(x, want)
