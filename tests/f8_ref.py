"""8-bit floating point with block scales by its definition, in 64 bits (test infrastructure)."""
import numpy as np
import torch


def scale_exp(amax):
    """The least e >= -126 with amax <= 448 * 2^e, for a float64 tensor of finite values."""
    a = amax.cpu().numpy()
    e = np.full(a.shape, -126, np.int64)
    m, x = np.frexp(a)  # a = m 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    want = np.where(m <= 0.875, x - 9, x - 8)
    return torch.from_numpy(np.where(a > 0, np.maximum(want, e), e))


def e4m3(v):
    """float64 values of at most 448 rounded to e4m3: four significant bits, steps of 2^-9 at least, to even."""
    _, x = torch.frexp(v)
    step = torch.exp2((x - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def quant(x, block=128):
    """(values, exponents) of the rows of x (M, K), float64 and int64 (M, ceil(K / block)); NaN where x is not finite."""
    x = x.detach().cpu().double()
    M, K = x.shape
    out = torch.empty_like(x)
    es = []
    for c in range(0, K, block):
        b = x[:, c:c + block]
        fin = torch.isfinite(b)
        e = scale_exp(torch.where(fin, b, torch.zeros_like(b)).abs().amax(1))
        es.append(e)
        s = torch.exp2(e.double())[:, None]
        out[:, c:c + block] = torch.where(fin, e4m3(torch.where(fin, b, torch.zeros_like(b)) / s) * s,
                                          torch.full_like(b, float("nan")))
    return out, torch.stack(es, 1)


def quant_stack(w, halves=1):
    """The values (E, K, N) of a stack with a scale per 128 x 128 block, float64."""
    w = w.detach().cpu().double()
    E, K, N = w.shape
    out = torch.empty_like(w)
    n = N // halves
    for e in range(E):
        for half in range(halves):
            for c in range(half * n, (half + 1) * n, 128):
                for k in range(0, K, 128):
                    b = w[e, k:k + 128, c:min(c + 128, (half + 1) * n)]
                    s = torch.exp2(scale_exp(b.abs().amax().reshape(1)).double())
                    out[e, k:k + 128, c:min(c + 128, (half + 1) * n)] = e4m3(b / s) * s
    return out


def counts_of(M, E, kind, seed=0):
    """Rows per expert summing to M: even, skewed with empty experts, or all in one."""
    g = np.random.default_rng(seed)
    if kind == "one":
        c = np.zeros(E, np.int64)
        c[E // 2] = M
    elif kind == "skew":
        p = 1.0 / np.arange(1, E + 1) ** 1.2
        p[E // 3] = 0 if E > 1 else 1
        c = g.multinomial(M, p / p.sum())
    else:
        c = np.full(E, M // E)
        c[: M % E] += 1
    return torch.from_numpy(c.astype(np.int32))
