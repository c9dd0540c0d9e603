"""Sorted rows past the counted ones, which exist where expert ids lie outside [0, E) (given ids, or a token whose router logits are
NaN): the index arrays mark them, and the backward neither reads nor writes through them."""
import pytest
import torch

from test_gpu_few import ops, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def some_ids(T, E, k, bad, dtype=torch.int32, seed=0):
    """Distinct experts per token, `bad` flat slots of which name none."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :k].contiguous()
    ok = ids.clone()
    at = torch.randperm(T * k, generator=g)[:bad]
    ids.view(-1)[at] = torch.tensor([-1, E, E + 5, 0x7FFFFFFF])[torch.arange(bad) % 4]
    dropped = torch.zeros(T * k, dtype=torch.bool)
    dropped[at] = True
    return ids.to(dtype).to(DEV), ok.to(dtype).to(DEV), dropped.to(DEV)


@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (300, 12, 3), (3000, 40, 2), (9000, 8, 2)])  # one workgroup; three passes
@pytest.mark.parametrize("rows", [False, True])  # (with the rows' copies: the pass by tokens)
@pytest.mark.parametrize("share", [0.0, 0.1, 1.0])
def test_dispatch_marks_them(T, E, k, rows, share):
    o = ops()
    n = round(share * T * k)
    for dtype in (torch.int32, torch.int64):
        ids, _, dropped = some_ids(T, E, k, n, dtype)
        for _ in range(2):
            torch.full((T * k,), 7, dtype=torch.int32, device=DEV)  # (what the arrays' memory may hold before)
            d = o.dispatch(ids, E, topk_w=torch.rand(T, k, device=DEV) + 0.5, x=rand(T, 64) if rows else None)
            M = T * k - n
            assert int(d.n_invalid) == n
            assert (d.order[M:] == -1).all() and (d.a_idx[M:] == -1).all() and (d.w_sorted[M:] == 0).all()
            assert torch.equal(d.order[:M].sort()[0].long(), torch.nonzero(~dropped).flatten())
            assert torch.equal(d.a_idx[:M], d.order[:M] // k) and (d.w_sorted[:M] > 0).all()


@pytest.mark.parametrize("T,E,k,d,h", [(70, 5, 2, 64, 48), (700, 6, 3, 128, 264), (5000, 8, 2, 64, 64)])
def test_backward_operators(T, E, k, d, h):
    """Slots that name no expert get a zero gradient of their weight, and the others the bits they have where every slot counts."""
    o = ops()
    M = T * k
    ids, ok, dropped = some_ids(T, E, k, M // 9)
    tw = torch.rand(T, k, device=DEV) + 0.5
    x, dout = rand(T, d, seed=1), rand(T, d, seed=2)
    wgu, wd = rand(E, d, 2 * h, seed=3, std=d ** -0.5), rand(E, h, d, seed=4, std=h ** -0.5)

    def run(ids):
        disp = o.dispatch(ids, E, topk_w=tw, x=x)
        n = int(disp.counts.sum())
        gu = o.grouped_mm(disp.xs, wgu, disp.counts, M)
        act, kept = o.swiglu_pack(gu)
        _, yhat = o.down_scatter(act, wd, disp.counts, M, disp.w_sorted, disp.order, keep_yhat=True)
        dys, dtw = o.combine_bwd(dout, yhat, disp, k)
        dys2, none = o.combine_bwd(dout, None, disp, k)
        assert none is None and torch.equal(dys[:n], dys2[:n])
        dgu, dtw2 = o.down_dgrad_swiglu_dw(dout, wd, disp.counts, M, gu, disp.order, k, a_idx=disp.a_idx, w_sorted=disp.w_sorted)
        dh = o.down_dgrad(dout, wd, disp.counts, M, a_idx=disp.a_idx)
        dgu3, _, dtw3 = o.swiglu_pack_bwd(dh, kept, disp.w_sorted, disp.order)
        flat = disp.order[:n].long()
        by_slot = []
        for t in (dys, dgu, dgu3):
            full = torch.zeros(M, t.shape[1], device=DEV, dtype=t.dtype)
            full[flat] = t[:n]
            by_slot.append(full)
        return (dtw.view(-1), dtw2.view(-1), dtw3), by_slot

    got, rows = run(ids)
    want, rows_ok = run(ok)
    for a, b in zip(got, want):
        assert (a[dropped] == 0).all() and torch.equal(a[~dropped], b[~dropped])
    for a, b in zip(rows, rows_ok):
        assert torch.equal(a[~dropped], b[~dropped])


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("T,E,k", [(5, 4, 2), (600, 10, 3), (5000, 8, 2)])
def test_training_on_a_nan_token(T, E, k, checkpoint):
    """A NaN token makes its own gradient and the weights' NaN; the other tokens' stays what it is without it."""
    from trenowanie_generatora_obrazkow_amd import moe_swiglu
    d, h, bad = 64, 48, T // 2
    wr, wgu, wd = rand(E, d, seed=5, std=d ** -0.5), rand(E, d, 2 * h, seed=3, std=d ** -0.5), rand(E, h, d, seed=4, std=h ** -0.5)
    x, dout = rand(T, d, seed=1), rand(T, d, seed=2)
    x2 = x.clone()
    x2[bad, 3] = float("nan")

    def run(x):
        leaves = [t.detach().clone().requires_grad_() for t in (x, wr, wgu, wd)]
        out, ids, tw = moe_swiglu(*leaves, k, checkpoint=checkpoint)
        (out * dout).sum().backward(retain_graph=True)
        (tw * tw.detach().nan_to_num()).sum().backward()
        return out.detach(), ids, [t.grad for t in leaves]

    out, _, grads = run(x)
    out2, ids2, grads2 = run(x2)
    assert ids2[bad, 0] == 0 and (ids2[bad, 1:] >= E).all()
    keep = torch.arange(T, device=DEV) != bad
    assert torch.equal(out2[keep], out[keep]) and torch.isnan(out2[bad]).all()
    assert torch.equal(grads2[0][keep], grads[0][keep]) and torch.isnan(grads2[0][bad]).all()
    assert torch.isnan(grads2[1]).any() and torch.isnan(grads2[2][0]).any() and torch.isnan(grads2[3][0]).any()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_residual_block_on_a_nan_token(checkpoint):
    from trenowanie_generatora_obrazkow_amd import MoEResidual
    torch.manual_seed(0)
    m = MoEResidual(64, 48, 6, 2, post_norm=True, device=DEV, checkpoint=checkpoint)
    x = rand(2, 20, 64)
    x[1, 7, 5] = float("nan")
    x.requires_grad_()
    out = m(x)
    out.sum().backward()
    at = torch.zeros(2, 20, dtype=torch.bool, device=DEV)
    at[1, 7] = True
    assert torch.equal(torch.isnan(out).all(-1), at) and torch.isfinite(out[~at]).all()
    assert torch.isnan(x.grad[at]).all() and torch.isfinite(x.grad[~at]).all()
