"""Tensor-level wrappers of the hmoe C entry points.  Each allocates its outputs with torch (caching allocator),
validates layouts, and launches on the current stream of the tensors' device.  GPU tensors only."""
from __future__ import annotations

from array import array
from dataclasses import dataclass

import torch

from . import _lib as L


def _dev_stream(t):
    L.require_gpu(t, "input")
    return L.stream(t.device)


_SIDE_STREAMS = {}  # device index -> side stream (kept off the modules, which may be copied or pickled)


def side_stream(device: torch.device):
    """One side stream per device for work that overlaps the main stream's, created with the default priority."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _SIDE_STREAMS:
        _SIDE_STREAMS[key] = torch.cuda.Stream(device=key)
    return _SIDE_STREAMS[key]


_SIDE_EVENTS = {}  # device index -> (fork, join) events of every hmoe_moe_block call


def side_events(device: torch.device):
    """A (fork, join) pair of events per device for forking work onto the side stream and joining it back: one pair
    serves every fork of every thread (wait_stream would make a new event each time), so a record and the wait on it must
    be one step under a lock, as hmoe_moe_block does it."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _SIDE_EVENTS:
        pair = (torch.cuda.Event(), torch.cuda.Event())
        for ev in pair:  # an event's handle exists from its first record on
            ev.record(torch.cuda.current_stream(key))
        _SIDE_EVENTS[key] = pair
    return _SIDE_EVENTS[key]


# Optional event probe: when `probe` is set to {op name: list}, each listed op records a (start, end) pair of
# torch.cuda.Events on the stream its kernels are launched on (the current stream) around its C call.
probe = None


class _Probe:
    def __init__(self, name):
        self.name = name
        self.ev = None

    def __enter__(self):
        if probe is not None and self.name in probe:
            self.ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
            self.ev[0].record()
        return self

    def __exit__(self, *exc):
        if self.ev is not None:
            self.ev[1].record()
            probe[self.name].append(self.ev)
        return False


def _contig(t, name):
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _need(t, name, shape=None, dtypes=None, contig=True, min_rows=None):
    """Validate a tensor handed to a C entry point: the kernels trust the sizes they are given, so a wrong shape,
    dtype or layout must stop here rather than become an out-of-range access on the device.  shape entries of None
    are not checked; min_rows: at least that many rows (a gathered operand); a row-strided 2-D tensor passes when
    contig=False as long as its rows are contiguous."""
    if t is None:
        raise ValueError(f"{name} is required")
    L.require_gpu(t, name)
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if shape is not None:
        if t.dim() != len(shape) or any(want is not None and got != want for got, want in zip(t.shape, shape)):
            raise ValueError(f"{name}: shape {tuple(t.shape)} does not match {shape}")
    if min_rows is not None and t.shape[0] < min_rows:
        raise ValueError(f"{name}: {t.shape[0]} rows, at least {min_rows} needed")
    if contig and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if not contig and t.dim() == 2 and t.stride(1) != 1:
        raise ValueError(f"{name} rows must be contiguous")
    return t


_BF16 = (torch.bfloat16,)
_H16 = (torch.bfloat16, torch.float16)  # the activation types of the forward kernels
_I32 = (torch.int32,)


def _act_dtype(t, name):
    """The 16-bit activation type of a forward call (bf16 or fp16), as the C code of the entry points' dtype."""
    if t.dtype not in _H16:
        raise TypeError(f"{name}: the hmoe forward kernels take bf16 or fp16 activations (got {t.dtype})")
    return L.dt(t)



def _rows_index(idx, name, M):
    return None if idx is None else _need(idx, name, (M,), _I32)


def _router_args(x, wr):
    if x.dim() != 2 or wr.dim() != 2 or x.dtype != torch.bfloat16 or wr.dtype != torch.bfloat16:
        raise TypeError("router expects a bf16 (T, d) x and a bf16 (E, d) weight")
    if wr.shape[1] != x.shape[1]:
        raise ValueError(f"router weight {tuple(wr.shape)} does not match x of width {x.shape[1]}")
    if x.stride(1) != 1:
        raise ValueError("x rows must be contiguous")
    L.require_gpu(wr, "router weight")


def route_topk(x: torch.Tensor, wr: torch.Tensor, k: int, bias=None, renorm=True, scaling=1.0, want_logits=True):
    """Softmax top-k router -> (logits (T, E) fp32 or None, topk_ids (T, k) int32, topk_w (T, k) fp32)."""
    T, d = x.shape
    E = wr.shape[0]
    _router_args(x, wr)
    wr = _contig(wr, "router weight")
    if bias is not None:
        if tuple(bias.shape) != (E,):
            raise ValueError(f"logit bias: shape {tuple(bias.shape)}, expected ({E},)")
        bias = _contig(bias.to(torch.float32), "bias")
    s = _dev_stream(x)
    # above 16 experts the logits buffer is passed even when not wanted: small token counts route through it
    logits = torch.empty(T, E, device=x.device, dtype=torch.float32) if want_logits or E > 16 else None
    ids = torch.empty(T, k, device=x.device, dtype=torch.int32)
    w = torch.empty(T, k, device=x.device, dtype=torch.float32)
    with _Probe("route_topk"):
        L.call("hmoe_route_topk", L.ptr(x), x.stride(0), L.ptr(wr), L.ptr(bias), T, d, E, k, int(bool(renorm)),
               float(scaling), L.ptr(logits), L.ptr(ids), L.ptr(w), s)
    return (logits if want_logits else None), ids, w


def moe_forward(x, wr, wgu, wd, k, bias=None, renorm=True, scaling=1.0, want_logits=False):
    """The routed forward of a layer in one C call (hmoe_moe_forward): route_topk, routed_gate_up, down_scatter and
    combine, with the same outputs and their intermediates in one workspace, for callers whose host time per layer
    matters (small batches).  x (T, d) bf16 with contiguous rows; wr (E, d), wgu (E, d, 2h), wd (E, h, d) bf16,
    contiguous; bias (E,) or None -> (out (T, d) bf16, topk_ids (T, k) int32, topk_w (T, k) fp32, logits (T, E)
    fp32 or None)."""
    T, d = x.shape
    E = wr.shape[0]
    _router_args(x, wr)
    _need(wr, "router weight", (E, d), _BF16)
    if wgu.dim() != 3 or wd.dim() != 3:
        raise ValueError("wgu (E, d, 2h) and wd (E, h, d) expected")
    h = wd.shape[1]
    _need(wgu, "wgu", (E, d, 2 * h), _BF16)
    _need(wd, "wd", (E, h, d), _BF16)
    if bias is not None:
        if tuple(bias.shape) != (E,):
            raise ValueError(f"logit bias: shape {tuple(bias.shape)}, expected ({E},)")
        bias = _contig(bias.to(torch.float32), "bias")
    if probe is not None and any(n in probe for n in _FWD_OPS):
        # event timing of single ops (bench.py's probe) needs the launches apart: the same entry points one by one
        logits, ids, w = route_topk(x, wr, k, bias=bias, renorm=renorm, scaling=scaling, want_logits=want_logits)
        disp, act, _ = routed_gate_up(x, ids, E, wgu, topk_w=w, want_inv=True)
        y, _ = down_scatter(act, wd, disp.counts, T * k, disp.w_sorted, disp.order)
        return combine(y, T, k, inv_pos=disp.inv_pos), ids, w, logits
    lib = L.lib()
    ws_bytes = lib.hmoe_moe_forward_workspace_size(T, d, E, k, h)
    if ws_bytes == 0:
        raise ValueError(f"moe_forward: unsupported sizes T={T} d={d} E={E} k={k} h={h}")
    dev = x.device
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    out = torch.empty(T, d, device=dev, dtype=torch.bfloat16)
    ids = torch.empty(T, k, device=dev, dtype=torch.int32)
    w = torch.empty(T, k, device=dev, dtype=torch.float32)
    logits = torch.empty(T, E, device=dev, dtype=torch.float32) if want_logits else None
    with _Probe("moe_forward"):
        L.call("hmoe_moe_forward", L.ptr(x), x.stride(0), L.ptr(wr), L.ptr(bias), L.ptr(wgu), L.ptr(wd), T, d, E, k,
               h, int(bool(renorm)), float(scaling), L.ptr(out), L.ptr(ids), L.ptr(w), L.ptr(logits), L.ptr(ws),
               ws_bytes, _dev_stream(x))
    return out, ids, w, logits


_FWD_OPS = ("route_topk", "dispatch", "gate_up_swiglu", "down_scatter", "combine")


def moe_experts(x, ids, tw, wgu, wd, wgu_s=None, wd_s=None):
    """The expert part of a forward whose routing the caller's gate decided, in one C call (hmoe_moe_experts):
    routed_gate_up (with inv_pos) and down_scatter with the same outputs.  x (T, d) bf16 or fp16 with contiguous rows;
    ids (T, k) int32 / int64; tw (T, k); wgu (E, d, 2h) and wd (E, h, d) of x's type, or int8 with scales wgu_s
    (E, 2h) and wd_s (E, d) -> (y (T*k, d) in (token, slot) order, inv_pos (T*k,) int32, n_invalid (1,) int32); the
    combine (with inv_pos) sums y over the slots.  wgu and wd may be F8Stacks (of 2 halves and of one): x and the activation
    are then quantised to 8 bits on the way, and the routing weights are not rounded."""
    if isinstance(wgu, F8Stack) or isinstance(wd, F8Stack):
        if wgu_s is not None or wd_s is not None:
            raise ValueError("F8Stacks hold their own scales")
        return _moe_experts_f8(x, ids, tw, wgu, wd)
    T, k = ids.shape
    if probe is not None and any(n in probe for n in _FWD_OPS):
        # event timing of single ops (bench.py's probe): the same entry points one by one
        disp, act, _ = routed_gate_up(x, ids, wgu.shape[0], wgu, topk_w=tw, wgu_s=wgu_s, want_inv=True)
        y, _ = down_scatter(act, wd, disp.counts, T * k, disp.w_sorted, disp.order, wd_s=wd_s)
        return y, disp.inv_pos, disp.n_invalid
    if x.dim() != 2 or x.shape[0] != T or x.stride(1) != 1:
        raise ValueError(f"x must be a ({T}, d) matrix with contiguous rows (got {tuple(x.shape)})")
    dt = _act_dtype(x, "x")
    d = x.shape[1]
    if wgu.dim() != 3 or wd.dim() != 3 or wgu.dtype not in (x.dtype, torch.int8) or wd.dtype != wgu.dtype:
        raise TypeError(f"wgu (E, d, 2h) and wd (E, h, d) of x's type or int8 expected (got {wgu.dtype}, {wd.dtype})")
    E, h = wgu.shape[0], wd.shape[1]
    L.require_gpu(x, "x")
    _need(ids, "topk_ids", (T, k), (torch.int32, torch.int64))
    if tuple(tw.shape) != (T, k):
        raise ValueError(f"topk_weight: shape {tuple(tw.shape)}, expected {(T, k)}")
    tw = _contig(tw if tw.dtype in (torch.float32, torch.bfloat16, torch.float16) else tw.float(), "topk_weight")
    _need(wgu, "wgu", (E, d, 2 * h), (wgu.dtype,))
    _need(wd, "wd", (E, h, d), (wd.dtype,))
    wgu_s = _w_scale(wgu, wgu_s, 2 * h)
    wd_s = _w_scale(wd, wd_s, d)
    w_dt = L.dt(wgu)
    lib = L.lib()
    ws_bytes = lib.hmoe_moe_experts_workspace_size(T, d, E, k, h, w_dt, dt)
    if ws_bytes == 0:
        raise ValueError(f"moe_experts: unsupported sizes T={T} d={d} E={E} k={k} h={h}")
    dev = x.device
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    y = torch.empty(T * k, d, device=dev, dtype=x.dtype)
    inv = torch.empty(T * k, device=dev, dtype=torch.int32)
    n_invalid = torch.empty(1, device=dev, dtype=torch.int32)
    L.call("hmoe_moe_experts", L.ptr(x), x.stride(0), L.ptr(ids), L.dt(ids), L.ptr(tw), L.dt(tw), L.ptr(wgu),
           L.ptr(wgu_s), L.dt(wgu_s) if wgu_s is not None else 0, L.ptr(wd), L.ptr(wd_s),
           L.dt(wd_s) if wd_s is not None else 0, w_dt, T, d, E, k, h, L.ptr(y), L.ptr(inv), L.ptr(n_invalid),
           L.ptr(ws), ws_bytes, dt, _dev_stream(x))
    return y, inv, n_invalid


def moe_block(x, gate_w, gate_b, k, n_group, topk_group, scaling, wgu, wgu_s, wd, wd_s, sh_wgu, sh_wd, sh_count,
              overlap=True):
    """The BailingMoeV2 block in one C call (hmoe_moe_block): route_sigmoid_group, moe_experts, the shared expert's
    gate_up_swiglu and down_scatter (overlap: on the side stream), and the combine with its output, with the same
    bits.  x (T, d) bf16 contiguous, T > 0; gate_w (E, d) bf16, gate_b (E,) fp32; wgu / wd bf16 or int8 with scales; sh_wgu
    (1, d, 2h'), sh_wd (1, h', d) bf16; sh_count (1,) int32 = T -> out (T, d) bf16."""
    T, d = x.shape
    E = gate_w.shape[0]
    _router_args(x, gate_w)
    _need(gate_w, "router weight", (E, d))
    _need(gate_b, "expert bias", (E,), (torch.float32,))
    if wgu.dim() != 3 or wd.dim() != 3 or wgu.dtype not in (torch.bfloat16, torch.int8) or wd.dtype != wgu.dtype:
        raise TypeError(f"wgu (E, d, 2h) and wd (E, h, d) of x's type or int8 expected (got {wgu.dtype}, {wd.dtype})")
    h, sh = wd.shape[1], sh_wd.shape[1]
    L.require_gpu(x, "x")
    _need(wgu, "wgu", (E, d, 2 * h))
    _need(wd, "wd", (E, h, d))
    wgu_s = _w_scale(wgu, wgu_s, 2 * h)
    wd_s = _w_scale(wd, wd_s, d)
    _need(sh_wgu, "shared gate/up", (1, d, 2 * sh), _BF16)
    _need(sh_wd, "shared down", (1, sh, d), _BF16)
    if sh_count is None or sh_count.dtype is not torch.int32 or sh_count.shape != (1,) or not sh_count.is_cuda:
        _need(sh_count, "shared row count", (1,), _I32)  # raises (called for every block it costs 1 us of about 80)
    w_dt = L.dt(wgu)
    ws_bytes = L.lib().hmoe_moe_block_workspace_size(T, d, E, k, h, sh, w_dt)
    if ws_bytes == 0:
        raise ValueError(f"moe_block: unsupported sizes T={T} d={d} E={E} k={k} h={h} shared={sh}")
    dev = x.device
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    out = torch.empty(T, d, device=dev, dtype=torch.bfloat16)
    side = fork = join = None
    if overlap:
        fork_ev, join_ev = side_events(dev)
        side, fork, join = side_stream(dev).cuda_stream, fork_ev.cuda_event, join_ev.cuda_event
    L.call("hmoe_moe_block", L.ptr(x), x.stride(0), L.ptr(gate_w), L.ptr(gate_b), n_group, topk_group, float(scaling),
           L.ptr(wgu), L.ptr(wgu_s), L.dt(wgu_s) if wgu_s is not None else 0, L.ptr(wd), L.ptr(wd_s),
           L.dt(wd_s) if wd_s is not None else 0, w_dt, L.ptr(sh_wgu), L.ptr(sh_wd), L.ptr(sh_count), sh, T, d, E, k, h,
           L.ptr(out), L.ptr(ws), ws_bytes, _dev_stream(x), side, fork, join)
    return out


def route_sigmoid_group(x: torch.Tensor, wr: torch.Tensor, k: int, n_group: int, topk_group: int, expert_bias=None,
                        scaling=1.0, want_scores=False):
    """BailingMoeV2 sigmoid, group-limited router -> (scores (T, E) fp32 or None, topk_ids (T, k) int32,
    topk_w (T, k) fp32)."""
    T, d = x.shape
    E = wr.shape[0]
    _router_args(x, wr)
    wr = _contig(wr, "router weight")
    if expert_bias is not None:
        if tuple(expert_bias.shape) != (E,):
            raise ValueError(f"expert bias: shape {tuple(expert_bias.shape)}, expected ({E},)")
        expert_bias = _contig(expert_bias.to(torch.float32), "expert bias")
    s = _dev_stream(x)
    # the scores buffer is passed even when not wanted: small token counts route through it (two launches that
    # spread the work over the chip)
    scores = torch.empty(T, E, device=x.device, dtype=torch.float32)
    ids = torch.empty(T, k, device=x.device, dtype=torch.int32)
    w = torch.empty(T, k, device=x.device, dtype=torch.float32)
    with _Probe("route_topk"):
        L.call("hmoe_route_sigmoid_group", L.ptr(x), x.stride(0), L.ptr(wr), L.ptr(expert_bias), T, d, E, k, n_group,
               topk_group, float(scaling), L.ptr(scores), L.ptr(ids), L.ptr(w), s)
    return (scores if want_scores else None), ids, w


@dataclass
class Dispatch:
    counts: torch.Tensor  # (E,) int32
    counts64: torch.Tensor  # (E,) int64 or None
    starts: torch.Tensor  # (E+1,) int32
    order: torch.Tensor  # (M,) int32  (= y_idx), -1 past the counted rows
    a_idx: torch.Tensor  # (M,) int32, -1 past the counted rows
    inv_pos: torch.Tensor  # (M,) int32
    w_sorted: torch.Tensor  # (M,) bf16 or None, 0 past the counted rows
    xs: torch.Tensor  # (M, d) bf16 or None
    xs_tiles: torch.Tensor = None  # the sorted rows as row-group tiles (bf16 storage) or None
    n_invalid: torch.Tensor = None  # (1,) int32 on the device: flat rows whose expert id lies outside [0, E)


def dispatch(topk_ids: torch.Tensor, E: int, topk_w=None, x=None, want_counts64=False, want_inv=True,
             want_xs=True, want_tiles=False, dtype=None) -> Dispatch:
    """Stable counting sort of the flat routed rows (aurora/hf_compat.py:69-72, 78, 80) and optionally, with x, the
    row permutation xs = x[a_idx] (want_xs) and the same rows as row-group tiles for gate_up_swiglu_tiles
    (want_tiles).  Expert ids outside [0, E) route nowhere (inv_pos -1, counted in no expert); their number is left
    on the device in n_invalid, read without a host sync only when the caller asks.  The sorted routing weights (and
    the copied rows) have x's type, bf16 or fp16 (dtype without x; bf16 by default)."""
    T, k = topk_ids.shape
    M = T * k
    dev = topk_ids.device
    s = _dev_stream(topk_ids)
    ids = _need(topk_ids, "topk_ids", (T, k), (torch.int32, torch.int64))
    if topk_w is not None:
        if tuple(topk_w.shape) != (T, k):
            raise ValueError(f"topk_weight: shape {tuple(topk_w.shape)}, expected {(T, k)}")
        topk_w = _contig(topk_w, "topk_weight")
        if topk_w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            topk_w = topk_w.float()
    if x is not None:
        dtype = x.dtype
    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in _H16:
        raise TypeError(f"dispatch: activations must be bf16 or fp16 (got {dtype})")
    counts = torch.empty(E, device=dev, dtype=torch.int32)
    counts64 = torch.empty(E, device=dev, dtype=torch.int64) if want_counts64 else None
    starts = torch.empty(E + 1, device=dev, dtype=torch.int32)
    order = torch.empty(M, device=dev, dtype=torch.int32)
    a_idx = torch.empty(M, device=dev, dtype=torch.int32)
    inv = torch.empty(M, device=dev, dtype=torch.int32) if want_inv else None
    w_sorted = torch.empty(M, device=dev, dtype=dtype) if topk_w is not None else None
    n_invalid = torch.empty(1, device=dev, dtype=torch.int32)
    xs = tiles = None
    d = 0
    ldx = 0
    if x is not None:
        _need(x, "x", (T, None), _H16, contig=False)  # xs = x[a_idx] reads rows a_idx < T
        d = x.shape[1]
        ldx = x.stride(0)
        if want_xs:
            xs = torch.empty(M, d, device=dev, dtype=dtype)
        if want_tiles:
            tiles = torch.empty(L.lib().hmoe_xs_tiles_bytes(M, E, d) // 2, device=dev, dtype=dtype)
    ws_bytes = L.lib().hmoe_dispatch_workspace_size(T, k, E)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with _Probe("dispatch"):
        L.call("hmoe_dispatch_tiles", L.ptr(ids), L.dt(ids), L.ptr(topk_w), L.dt(topk_w) if topk_w is not None else 0,
               T, k, E, L.ptr(x), ldx, d, L.ptr(xs), L.ptr(tiles), L.ptr(counts), L.ptr(counts64), L.ptr(starts),
               L.ptr(order), L.ptr(a_idx), L.ptr(inv), L.ptr(w_sorted), L.ptr(n_invalid), L.ptr(ws), ws_bytes,
               L.dt(dtype), s)
    return Dispatch(counts, counts64, starts, order, a_idx, inv, w_sorted, xs, tiles, n_invalid)


def make_schedule(counts: torch.Tensor, M: int, block_m: int = 64):
    E = counts.numel()
    nb = -(-M // block_m) + E
    s = _dev_stream(counts)
    counts = _contig(counts, "counts")
    if counts.dtype not in (torch.int32, torch.int64):
        counts = counts.to(torch.int64)
    out = [torch.empty(nb, device=counts.device, dtype=torch.int32) for _ in range(3)]
    with _Probe("make_schedule"):
        L.call("hmoe_make_schedule", L.ptr(counts), L.dt(counts), E, M, block_m, *(L.ptr(o) for o in out), s)
    return tuple(out)


def _counts(counts, E):
    """Rows per expert, (E,) int32 or int64 on the GPU: the kernels read E entries."""
    if counts.dtype not in (torch.int32, torch.int64):
        counts = counts.to(torch.int64)
    return _need(counts, "counts", (E,), (torch.int32, torch.int64))


def grouped_mm(a, w, counts, M, a_idx=None, y_idx=None, scale=None, w_scale=None, out=None):
    """y[y_idx[r] or r] = (a[a_idx[r] or r] @ w[e(r)]) * w_scale[e(r)] * scale[r], y (M, N) bf16.  The index
    values are trusted (in range: a_idx < rows of a, y_idx < M); everything else is checked here."""
    if w.dim() != 3 or w.dtype not in (a.dtype, torch.int8):
        raise TypeError(f"w must be an (E, K, N) stack of a's type or int8 (got {tuple(w.shape)} {w.dtype})")
    E, K, N = w.shape
    s = _dev_stream(a)
    _act_dtype(a, "a")
    counts = _counts(counts, E)
    if a.stride(1) != 1:
        a = a.contiguous()
    if w.stride(2) != 1:
        w = w.contiguous()
    a_idx = _rows_index(a_idx, "a_idx", M)
    y_idx = _rows_index(y_idx, "y_idx", M)
    _need(a, "a", (None, K), _H16, contig=False, min_rows=min(1, M) if a_idx is not None else M)
    if a_idx is not None and a.shape[0] * a.stride(0) * 2 >= 2 ** 31:
        raise ValueError("a gathered through a_idx must span less than 2 GiB (32-bit row offsets)")
    if w_scale is not None:
        w_scale = _contig(w_scale, "w_scale")
        if w_scale.shape != (E, N):
            raise ValueError(f"w_scale must be (E, N) = {(E, N)}, got {tuple(w_scale.shape)}")
    if out is not None:
        _need(out, "out", (M, N), (a.dtype,), contig=False)
    y = out if out is not None else torch.empty(M, N, device=a.device, dtype=a.dtype)
    if scale is not None:
        scale = _contig(scale, "scale")
        if scale.dtype not in (a.dtype, torch.float32):
            scale = scale.float()
        _need(scale, "scale", (M,))
    with _Probe("grouped_mm"):
        L.call("hmoe_grouped_mm", L.ptr(a), a.stride(0), L.dt(a), L.ptr(w), L.dt(w), E, K, N, w.stride(0), w.stride(1),
               L.ptr(counts), L.dt(counts), M, L.ptr(a_idx), L.ptr(y_idx), L.ptr(scale),
               L.dt(scale) if scale is not None else 0, L.ptr(w_scale), L.dt(w_scale) if w_scale is not None else 0,
               L.ptr(y), y.stride(0), s)
    return y


def _w_scale(w, w_s, n):
    """int8 weights need their (E, n) per-column scales; bf16 weights take none."""
    if (w.dtype == torch.int8) != (w_s is not None):
        raise ValueError("int8 weights come with a scale (E, N); bf16 weights take none")
    if w_s is not None:
        w_s = _contig(w_s, "weight scale")
        if w_s.shape != (w.shape[0], n) or w_s.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"weight scale must be bf16 or fp32 of shape {(w.shape[0], n)}")
    return w_s


def gate_up_swiglu(x, wgu, counts, M, a_idx=None, keep_gu=False, wgu_s=None):
    """act = bf16(bf16(silu(g)) * u) for [g | u] = x[a_idx] @ wgu[e]; wgu bf16, or int8 with per-column scales
    wgu_s (E, 2h) (inference only: no gu)."""
    if wgu.dim() != 3 or wgu.dtype not in (x.dtype, torch.int8) or wgu.shape[2] % 2:
        raise TypeError(f"wgu must be an (E, d, 2h) stack of x's type or int8 (got {tuple(wgu.shape)} {wgu.dtype})")
    E, d, h2 = wgu.shape
    h = h2 // 2
    s = _dev_stream(x)
    dt = _act_dtype(x, "x")
    wgu = _contig(wgu, "wgu")
    counts = _counts(counts, E)
    wgu_s = _w_scale(wgu, wgu_s, h2)
    a_idx = _rows_index(a_idx, "a_idx", M)
    _need(x, "x", (None, d), _H16, contig=False, min_rows=min(1, M) if a_idx is not None else M)
    act = torch.empty(M, h, device=x.device, dtype=x.dtype)
    if wgu_s is not None:
        if keep_gu:
            raise ValueError("int8 weights are inference only (no gu kept)")
        with _Probe("gate_up_swiglu"):
            L.call("hmoe_gate_up_swiglu_i8", L.ptr(x), x.stride(0), L.ptr(a_idx), L.ptr(wgu), L.ptr(wgu_s),
                   L.dt(wgu_s), E, d, h, L.ptr(counts), L.dt(counts), M, L.ptr(act), dt, s)
        return act, None
    gu = torch.empty(M, h2, device=x.device, dtype=x.dtype) if keep_gu else None
    with _Probe("gate_up_swiglu"):
        L.call("hmoe_gate_up_swiglu", L.ptr(x), x.stride(0), L.ptr(a_idx), L.ptr(wgu), E, d, h, L.ptr(counts),
               L.dt(counts), M, L.ptr(act), L.ptr(gu), dt, s)
    return act, gu


def gate_up_swiglu_tiles(xs_tiles, wgu, counts, M, keep_gu=False):
    """gate_up_swiglu on the row-group tiles a dispatch(want_tiles=True) wrote (16-bit weights of the tiles' type):
    identical act / gu."""
    if wgu.dim() != 3 or wgu.dtype != xs_tiles.dtype or wgu.shape[2] % 2:
        raise TypeError(f"wgu must be an (E, d, 2h) stack of the tiles' type (got {tuple(wgu.shape)} {wgu.dtype})")
    E, d, h2 = wgu.shape
    h = h2 // 2
    s = _dev_stream(xs_tiles)
    dt = _act_dtype(xs_tiles, "xs_tiles")
    wgu = _contig(wgu, "wgu")
    counts = _counts(counts, E)
    _need(xs_tiles, "xs_tiles", (L.lib().hmoe_xs_tiles_bytes(M, E, d) // 2,), _H16)
    act = torch.empty(M, h, device=xs_tiles.device, dtype=xs_tiles.dtype)
    gu = torch.empty(M, h2, device=xs_tiles.device, dtype=xs_tiles.dtype) if keep_gu else None
    with _Probe("gate_up_swiglu"):
        L.call("hmoe_gate_up_swiglu_tiles", L.ptr(xs_tiles), L.ptr(wgu), E, d, h, L.ptr(counts), L.dt(counts), M,
               L.ptr(act), L.ptr(gu), dt, s)
    return act, gu


# The tiles save about 7% of the gate/up GEMM (2 M d 2h flops) for M d 2 more bytes written by the dispatch, so
# they pay for wide hidden layers only.  Whole forward passes, same process: h = 4096 (C3) 1290 against 1297 us,
# h = 2048 (C2, 2048 tokens) 143 against 128, h = 320 (BailingMoeV2-like, bf16) 807 against 747.  Below this the
# GEMM gathers the rows itself.
TILES_MIN_H = 4096


def routed_gate_up(x, ids, E, wgu, topk_w=None, wgu_s=None, keep_gu=False, want_xs=False, want_inv=True):
    """dispatch + gate/up GEMM of the routed rows: with bf16 weights and a wide hidden layer the dispatch writes the
    rows as row-group tiles and the GEMM reads them (1 KB copies); otherwise (int8 weights, h below TILES_MIN_H,
    tiles past the GEMM's 32-bit offsets) the GEMM gathers the rows of x itself.  want_xs: also the row-major
    permuted copy (the gate/up weight gradient reads it).  Returns (Dispatch, act, gu)."""
    T, k = ids.shape
    M = T * k
    d = x.shape[1]
    h = wgu.shape[2] // 2
    tiles = (wgu_s is None and wgu.dtype == x.dtype and h >= TILES_MIN_H
             and L.lib().hmoe_xs_tiles_bytes(M, E, d) < (1 << 31))
    disp = dispatch(ids, E, topk_w=topk_w, x=x if (tiles or want_xs) else None, want_inv=want_inv, want_xs=want_xs,
                    want_tiles=tiles, dtype=x.dtype)
    if tiles:
        act, gu = gate_up_swiglu_tiles(disp.xs_tiles, wgu, disp.counts, M, keep_gu=keep_gu)
        disp.xs_tiles = None  # read once: not kept alive with the dispatch
    elif want_xs:
        act, gu = gate_up_swiglu(disp.xs, wgu, disp.counts, M, keep_gu=keep_gu, wgu_s=wgu_s)
    else:
        act, gu = gate_up_swiglu(x, wgu, disp.counts, M, a_idx=disp.a_idx, keep_gu=keep_gu, wgu_s=wgu_s)
    return disp, act, gu


def down_scatter(act, wd, counts, M, w_sorted, y_idx, keep_yhat=False, wd_s=None):
    """y[y_idx[r]] = bf16(act[r] @ wd[e] * w_sorted[r]); wd bf16, or int8 with per-column scales wd_s (E, d)."""
    if wd.dim() != 3 or wd.dtype not in (act.dtype, torch.int8):
        raise TypeError(f"wd must be an (E, h, d) stack of act's type or int8 (got {tuple(wd.shape)} {wd.dtype})")
    E, h, d = wd.shape
    s = _dev_stream(act)
    dt = _act_dtype(act, "act")
    wd = _contig(wd, "wd")
    counts = _counts(counts, E)
    wd_s = _w_scale(wd, wd_s, d)
    _need(act, "act", (M, h), _H16)
    y_idx = _rows_index(y_idx, "y_idx", M)
    if w_sorted is not None:
        _need(w_sorted, "w_sorted", (M,), (act.dtype,))
    y = torch.empty(M, d, device=act.device, dtype=act.dtype)
    if wd_s is not None:
        if keep_yhat:
            raise ValueError("int8 weights are inference only (no yhat kept)")
        with _Probe("down_scatter"):
            L.call("hmoe_down_scatter_i8", L.ptr(act), L.ptr(wd), L.ptr(wd_s), L.dt(wd_s), E, h, d, L.ptr(counts),
                   L.dt(counts), M, L.ptr(w_sorted), L.ptr(y_idx), L.ptr(y), dt, s)
        return y, None
    yhat = torch.empty(M, d, device=act.device, dtype=act.dtype) if keep_yhat else None
    with _Probe("down_scatter"):
        L.call("hmoe_down_scatter", L.ptr(act), L.ptr(wd), E, h, d, L.ptr(counts), L.dt(counts), M, L.ptr(w_sorted),
               L.ptr(y_idx), L.ptr(y), L.ptr(yhat), dt, s)
    return y, yhat


def combine(y, T, k, add=None, inv_pos=None):
    """out[t] = bf16(sum_j y[t*k + j]) (+ add[t], rounded once more: bf16 + bf16).  inv_pos (T*k,) from the dispatch:
    slots routed nowhere (inv_pos < 0: an expert id outside [0, E)) add zeros instead of their unwritten rows."""
    d = y.shape[1]
    _need(y, "y", (T * k, d), _H16)
    dt = _act_dtype(y, "y")
    inv_pos = _rows_index(inv_pos, "inv_pos", T * k)
    out = torch.empty(T, d, device=y.device, dtype=y.dtype)
    with _Probe("combine"):
        if add is None:
            L.call("hmoe_combine", L.ptr(_contig(y, "y")), L.ptr(inv_pos), T, k, d, L.ptr(out), dt, _dev_stream(y))
        else:
            if add.shape != (T, d) or add.dtype != y.dtype:
                raise ValueError(f"add must be {y.dtype} of shape {(T, d)}")
            L.call("hmoe_combine_add", L.ptr(_contig(y, "y")), L.ptr(inv_pos), T, k, d, L.ptr(_contig(add, "add")),
                   L.ptr(out), dt, _dev_stream(y))
    return out


def combine_bwd(dout, yhat, disp: Dispatch, k):
    """(dys (M, d) bf16, dtopk_w (T, k) fp32): the routing-weighted upstream rows in sorted order and, with yhat
    (the unscaled down-projection rows, sorted), <dout[t], yhat[r]>; yhat None: (dys, None).  Rows of dys past the counted
    ones are not written; dtopk_w is 0 for a slot whose id names no expert."""
    T, d = dout.shape
    M = T * k
    dout = dout.contiguous()
    if yhat is not None:
        _need(yhat, "yhat", (M, d), _BF16)
    _need(dout, "dout", (T, d), _BF16)
    for t_, n_ in ((disp.order, "order"), (disp.a_idx, "a_idx")):
        _need(t_, n_, (M,), _I32)
    _need(disp.w_sorted, "w_sorted", (M,), _BF16)
    dys = torch.empty(M, d, device=dout.device, dtype=torch.bfloat16)
    dtw = torch.zeros(T, k, device=dout.device, dtype=torch.float32) if yhat is not None else None  # (0 for slots without a row)
    with _Probe("combine_bwd"):
        L.call("hmoe_combine_bwd", L.ptr(dout), L.ptr(yhat), L.ptr(disp.order), L.ptr(disp.a_idx), L.ptr(disp.w_sorted),
               M, k, d, L.ptr(dys), L.ptr(dtw), _dev_stream(dout))
    return dys, dtw


def down_dgrad_swiglu(dy, wd, counts, M, gu, a_idx=None, w_sorted=None):
    """dgu (M, 2h) from the upstream gradient dy (T, d) gathered through a_idx (or sorted rows (M, d) when a_idx is
    None) and scaled by w_sorted in fp32."""
    _need(wd, "wd", (None, None, None), _BF16)
    E, h, d = wd.shape
    counts = _counts(counts, E)
    a_idx = _rows_index(a_idx, "a_idx", M)
    _need(dy, "dy", (None, d), _BF16, min_rows=min(1, M) if a_idx is not None else M)
    _need(gu, "gu", (M, 2 * h), _BF16)
    if w_sorted is not None:
        _need(w_sorted, "w_sorted", (M,), _BF16)
    dgu = torch.empty(M, 2 * h, device=dy.device, dtype=torch.bfloat16)
    with _Probe("down_dgrad_swiglu"):
        L.call("hmoe_down_dgrad_swiglu", L.ptr(dy), L.ptr(a_idx), L.ptr(w_sorted), L.ptr(wd), E, h, d, L.ptr(counts),
               L.dt(counts), M, L.ptr(gu), L.ptr(dgu), _dev_stream(dy))
    return dgu


def down_dgrad_swiglu_dw(dy, wd, counts, M, gu, order, k, a_idx=None, w_sorted=None):
    """(dgu, dtopk_w): down_dgrad_swiglu's dgu and, from the same product, the routing-weight gradient dtopk_w (T, k)
    fp32 = sum_n (dy[t] @ wd[e]^T)[n] * act[r][n], act recomputed from gu as the forward rounds it; 0 for a slot whose id
    names no expert."""
    _need(wd, "wd", (None, None, None), _BF16)
    E, h, d = wd.shape
    counts = _counts(counts, E)
    a_idx = _rows_index(a_idx, "a_idx", M)
    _need(dy, "dy", (None, d), _BF16, min_rows=min(1, M) if a_idx is not None else M)
    _need(gu, "gu", (M, 2 * h), _BF16)
    order = _rows_index(order, "order", M)
    if order is None:
        raise ValueError("order is required")
    if w_sorted is not None:
        _need(w_sorted, "w_sorted", (M,), _BF16)
    if M % k:
        raise ValueError(f"M = {M} is not a multiple of k = {k}")
    dgu = torch.empty(M, 2 * h, device=dy.device, dtype=torch.bfloat16)
    dtw = torch.zeros(M // k, k, device=dy.device, dtype=torch.float32)  # (slots without a row keep it)
    ws_bytes = L.lib().hmoe_down_dgrad_dw_workspace_size(M, h)
    ws = torch.empty(ws_bytes, device=dy.device, dtype=torch.uint8)
    with _Probe("down_dgrad_swiglu"):
        L.call("hmoe_down_dgrad_swiglu_dw", L.ptr(dy), L.ptr(a_idx), L.ptr(w_sorted), L.ptr(wd), E, h, d,
               L.ptr(counts), L.dt(counts), M, L.ptr(gu), L.ptr(dgu), L.ptr(order), L.ptr(dtw), L.ptr(ws), ws_bytes,
               _dev_stream(dy))
    return dgu, dtw


def down_dgrad(dy, wd, counts, M, a_idx=None):
    """dh (M, h) bf16 = dy[a_idx[r] or r] @ wd[e]^T, not scaled: the product of down_dgrad_swiglu alone."""
    _need(wd, "wd", (None, None, None), _BF16)
    E, h, d = wd.shape
    counts = _counts(counts, E)
    a_idx = _rows_index(a_idx, "a_idx", M)
    _need(dy, "dy", (None, d), _BF16, min_rows=min(1, M) if a_idx is not None else M)
    dh = torch.empty(M, h, device=dy.device, dtype=torch.bfloat16)
    with _Probe("down_dgrad"):
        L.call("hmoe_down_dgrad", L.ptr(dy), L.ptr(a_idx), L.ptr(wd), E, h, d, L.ptr(counts), L.dt(counts), M, L.ptr(dh),
               _dev_stream(dy))
    return dh


def dgrad_parts(M, wgu):
    """Parts the gate/up dgrad's reduction is best split into for M rows (1: not split)."""
    E, d, h2 = wgu.shape
    return L.lib().hmoe_gate_up_dgrad_parts(M, E, d, h2 // 2)


def gate_up_dgrad(dgu, wgu, counts, M, dtype=torch.float32, parts=1):
    """dxs (M, d) = dgu @ wgu[e]^T; parts > 1: (parts, M, d) fp32, the reduction split (unpermute_bwd adds the parts)."""
    _need(wgu, "wgu", (None, None, None), _BF16)
    E, d, h2 = wgu.shape
    counts = _counts(counts, E)
    _need(dgu, "dgu", (M, h2), _BF16)
    if parts > 1 and dtype != torch.float32:
        raise TypeError(f"a split dgrad is fp32 (got {dtype})")
    dxs = torch.empty((M, d) if parts == 1 else (parts, M, d), device=dgu.device, dtype=dtype)
    with _Probe("gate_up_dgrad"):
        if parts == 1:
            L.call("hmoe_gate_up_dgrad", L.ptr(dgu), L.ptr(wgu), E, d, h2 // 2, L.ptr(counts), L.dt(counts), M,
                   L.ptr(dxs), L.dt(dxs), _dev_stream(dgu))
        else:
            L.call("hmoe_gate_up_dgrad_split", L.ptr(dgu), L.ptr(wgu), E, d, h2 // 2, L.ptr(counts), L.dt(counts), M,
                   L.ptr(dxs), parts, _dev_stream(dgu))
    return dxs


def grouped_wgrad(a, b, counts, E, dtype=torch.bfloat16):
    M, P = a.shape
    N = b.shape[1]
    counts = _counts(counts, E)
    _need(a, "a", (M, P), _BF16, contig=False)
    _need(b, "b", (M, N), _BF16, contig=False)
    dw = torch.empty(E, P, N, device=a.device, dtype=dtype)
    with _Probe("grouped_wgrad"):
        L.call("hmoe_grouped_wgrad", L.ptr(a), a.stride(0), L.ptr(b), b.stride(0), E, P, N, L.ptr(counts), L.dt(counts), M,
               L.ptr(dw), L.dt(dw), _dev_stream(a))
    return dw


def router_bwd(logits, ids, dtw, x, renorm=True, scaling=1.0, dwr_dtype=torch.float32, want_dwr=True):
    T, E = logits.shape
    k = ids.shape[1]
    d = x.shape[1]
    _need(logits, "logits", (T, E), (torch.float32,))
    _need(ids, "topk_ids", (T, k), _I32)
    _need(dtw, "dtopk_w", (T, k), (torch.float32,))
    _need(x, "x", (T, d), _BF16, contig=False)
    dl = torch.empty(T, E, device=logits.device, dtype=torch.float32)
    dwr = torch.empty(E, d, device=logits.device, dtype=dwr_dtype) if want_dwr else None
    ws_bytes = L.lib().hmoe_router_bwd_workspace_size(T, E, d) if want_dwr else 0
    ws = torch.empty(max(ws_bytes, 1), device=logits.device, dtype=torch.uint8)
    with _Probe("router_bwd"):
        L.call("hmoe_router_bwd", L.ptr(logits), L.ptr(ids), L.ptr(dtw), T, E, k, int(bool(renorm)), float(scaling),
               L.ptr(x), x.stride(0), d, L.ptr(dl), L.ptr(dwr), L.dt(dwr_dtype), L.ptr(ws) if want_dwr else None, ws_bytes,
               _dev_stream(logits))
    return dl, dwr


def unpermute_bwd(dxs, inv_pos, T, k, dlogits=None, wr=None):
    """dx (T, d) bf16 from the sorted rows dxs (T*k, d), or the parts (parts, T*k, d) fp32 of a split gate_up_dgrad."""
    parts = dxs.shape[0] if dxs.dim() == 3 else 1
    d = dxs.shape[-1]
    E = wr.shape[0] if wr is not None else 0
    if dxs.dim() == 3:
        _need(dxs, "dxs", (None, T * k, d), (torch.float32,))
    else:
        _need(dxs, "dxs", (T * k, d), (torch.float32, torch.bfloat16))
    _need(inv_pos, "inv_pos", (T * k,), _I32)
    if (dlogits is None) != (wr is None):
        raise ValueError("dlogits and wr come together")
    if wr is not None:
        _need(wr, "wr", (E, d), _BF16)
        _need(dlogits, "dlogits", (T, E), (torch.float32,))
    dx = torch.empty(T, d, device=dxs.device, dtype=torch.bfloat16)
    with _Probe("unpermute_bwd"):
        if dxs.dim() == 3:
            L.call("hmoe_unpermute_bwd_split", L.ptr(dxs), parts, L.ptr(inv_pos), L.ptr(dlogits), L.ptr(wr), T, k, d, E,
                   L.ptr(dx), _dev_stream(dxs))
        else:
            L.call("hmoe_unpermute_bwd", L.ptr(dxs), L.dt(dxs), L.ptr(inv_pos), L.ptr(dlogits), L.ptr(wr), T, k, d, E,
                   L.ptr(dx), _dev_stream(dxs))
    return dx


# ---------------------------------------------------------------------------------------------------------------
# Routing from logits, the norms around the block, gradient clipping
# ---------------------------------------------------------------------------------------------------------------
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_SCORES = {"softmax": 0, "sigmoid": 1}


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call_on(dev, name, *args):
    """A C call with its stream, launched on `dev` also where another device is the current one."""
    i = dev.index
    f = _entry.get(name) or _entry.setdefault(name, getattr(L.lib(), name))
    if i == _current_device():
        rc = f(*args, L.stream(i))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, L.stream(i))
    if rc != 0:
        raise L.HmoeError(name, rc)


_entry = {}  # C entry points by name


def _on(t, name, dev, shape, dtypes):
    """A contiguous operand of a call whose first tensor lives on `dev`; None passes."""
    if t is None or (t.dtype in dtypes and t.shape == shape and t.is_contiguous() and t.device == dev):
        return t
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {dev}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _rows(t, name, dtypes=_FLOATS):
    """(T, d, row stride) of a matrix whose rows are contiguous."""
    if t.dim() != 2 or not t.is_cuda:
        L.require_gpu(t, name)
        raise ValueError(f"{name} must be a (rows, width) matrix (got {tuple(t.shape)})")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    T, d = t.shape
    if d % 8 or d == 0:
        raise ValueError(f"{name}: width {d} must be a positive multiple of 8")
    if t.is_contiguous():
        return T, d, d
    ld = t.stride(0) if T > 1 else d
    if t.stride(1) != 1 or ld < d or ld % 8:
        raise ValueError(f"{name}: rows must be contiguous, with a row stride of a multiple of 8 (strides {t.stride()})")
    return T, d, ld


def _routing(logits, k, score, n_group, topk_group, group_top):
    """(T, E, row stride) of logits, and every condition on the sizes."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _FLOATS:
        L.require_gpu(logits, "logits")
        raise TypeError(f"logits must be a (T, E) matrix of bf16, fp16 or fp32 (got {tuple(logits.shape)} {logits.dtype})")
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid' (got {score!r})")
    T, E = logits.shape
    if not 1 <= k <= E or k > 16 or E > 512:
        raise ValueError(f"routing takes up to 512 experts and 1 to min(16, E) slots (got E = {E}, k = {k})")
    ld = E
    if not logits.is_contiguous():
        ld = logits.stride(0) if T > 1 else E
        if (E > 1 and logits.stride(1) != 1) or ld < E:
            raise ValueError(f"logits rows must be contiguous (strides {logits.stride()})")
    if n_group != 1 or topk_group != 1 or group_top not in (1, 2):
        if n_group < 1 or not 1 <= topk_group <= n_group or E % n_group or group_top not in (1, 2):
            raise ValueError(f"groups: E = {E} must divide into n_group = {n_group}, 1 <= topk_group = {topk_group} <= "
                             f"n_group, group_top = {group_top} 1 or 2")
        if topk_group < n_group and (n_group > 64 or E // n_group < group_top or k > topk_group * (E // n_group)):
            raise ValueError(f"{topk_group} of {n_group} groups of {E // n_group} experts cannot give k = {k} (at most 64 "
                             f"groups)")
    return T, E, ld


def route_scores(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_top=2, renorm=True, scaling=1.0,
                 live=None):
    """The k experts of each token from given logits (T, E), bf16, fp16 or fp32 -> (topk_ids (T, k) int32, topk_w (T, k)
    fp32).  score "softmax" or "sigmoid"; bias (E,) fp32 joins the scores for the selection only; topk_group < n_group keeps
    the groups with the largest sums of their group_top best values; renorm divides the weights by their sum; live (T,)
    bool: padding tokens (False) get ids -1 and weights 0, which dispatch and moe_experts route nowhere -- for inference: the
    experts' backward (combine_bwd, down_dgrad_swiglu_dw) takes routings that name an expert for every slot, so a training
    step routes its padding too and gives it a zero gradient."""
    T, E, ld = _routing(logits, k, score, n_group, topk_group, group_top)
    dev = logits.device
    _on(bias, "bias", dev, (E,), (torch.float32,))
    _on(live, "live", dev, (T,), (torch.bool, torch.uint8))
    ids = torch.empty(T, k, device=dev, dtype=torch.int32)
    w = torch.empty(T, k, device=dev, dtype=torch.float32)
    _call_on(dev, "hmoe_route_scores", logits.data_ptr(), ld, L.dt(logits), L.ptr(bias), L.ptr(live), T, E, k,
             _SCORES[score], n_group, topk_group, group_top, int(bool(renorm)), float(scaling), ids.data_ptr(), w.data_ptr())
    return ids, w


def route_scores_bwd(dtw, tw, logits, ids, score="softmax", renorm=True, scaling=1.0):
    """dlogits (T, E) of the logits' type from dtw (T, k) fp32, the gradient of route_scores' weights tw; ids as it gave
    them."""
    T, k = ids.shape
    _, E, ld = _routing(logits, k, score, 1, 1, 1)
    dev = logits.device
    if logits.shape[0] != T:
        raise ValueError(f"topk_ids for {T} tokens, logits for {logits.shape[0]}")
    _on(ids, "topk_ids", dev, (T, k), _I32)
    _on(tw, "topk_w", dev, (T, k), (torch.float32,))
    _on(dtw, "dtopk_w", dev, (T, k), (torch.float32,))
    dl = torch.empty(T, E, device=dev, dtype=logits.dtype)
    _call_on(dev, "hmoe_route_scores_bwd", dtw.data_ptr(), tw.data_ptr(), logits.data_ptr(), ld, L.dt(logits),
             ids.data_ptr(), T, E, k, _SCORES[score], int(bool(renorm)), float(scaling), dl.data_ptr())
    return dl


def router_wgrad(dlogits, x, dtype=torch.float32):
    """dwr (E, d) = dlogits^T @ x from the logits' gradient (T, E) fp32 and x (T, d) bf16; fp32 or bf16."""
    T, E = dlogits.shape
    d = x.shape[1]
    _need(x, "x", (T, d), _BF16, contig=False)
    dev = x.device
    _on(dlogits, "dlogits", dev, (T, E), (torch.float32,))
    dwr = torch.empty(E, d, device=dev, dtype=dtype)
    ws_bytes = L.lib().hmoe_router_bwd_workspace_size(T, E, d)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _call_on(dev, "hmoe_router_wgrad", L.ptr(dlogits), L.ptr(x), x.stride(0), T, E, d, L.ptr(dwr), L.dt(dwr), L.ptr(ws),
             ws_bytes)
    return dwr


def _sample_params(T, d, dev, starts, a, a_name, b=None, b_name=""):
    """The number of samples B of per-sample parameters a and b: (B, d) each, or (d,) for one set; with starts (B + 1,)."""
    if a is None and b is None and starts is None:
        return 1
    B = None
    for t, name in ((a, a_name), (b, b_name)):
        if t is None:
            continue
        n = 1 if t.dim() == 1 else t.shape[0]
        _on(t, name, dev, (d,) if t.dim() == 1 else (n, d), _FLOATS)
        if B is not None and n != B:
            raise ValueError(f"{name} has {n} samples, another parameter {B}")
        B = n
    if starts is not None:
        n = starts.numel() - 1
        _on(starts, "starts", dev, (n + 1,), _I32)
        if n < 1 or (B is not None and B != n):
            raise ValueError(f"starts names {n} samples" + ("" if B is None else f", the parameters hold {B}"))
        return n
    if B < 1 or T % B:
        raise ValueError(f"{T} rows do not divide into {B} samples (pass starts for samples of unequal lengths)")
    return B


def _block_dtype(stream, dtype):
    if dtype is None or dtype is stream:
        return stream
    if dtype not in _FLOATS or stream is not torch.float32:
        raise TypeError(f"a block type of {dtype} does not go with a stream of {stream} (equal, or an fp32 stream)")
    return dtype


def _dt0(t):
    return 0 if t is None else L._DT[t.dtype]


def norm_modulate(x, weight=None, scale=None, shift=None, starts=None, eps=1e-6, dtype=None):
    """h (T, d) = n * weight * (1 + scale_b) + shift_b, n = x / sqrt(mean(x^2) + eps): the input of a block from the
    residual stream x (T, d).  weight (d,); scale and shift (B, d) per sample of T / B rows each, or with starts (B + 1,)
    int32 of rows starts[b] .. starts[b + 1] - 1 (rows outside are padding: h = 0); (d,) for one set.  dtype: h's type, x's
    by default; an fp32 stream may have a 16-bit block."""
    T, d, ldx = _rows(x, "x")
    dev = x.device
    dtype = _block_dtype(x.dtype, dtype)
    _on(weight, "weight", dev, (d,), _FLOATS)
    B = _sample_params(T, d, dev, starts, scale, "scale", shift, "shift")
    if scale is not None and shift is not None and scale.dtype != shift.dtype:
        raise TypeError(f"scale and shift must have one type (got {scale.dtype}, {shift.dtype})")
    h = torch.empty(T, d, device=dev, dtype=dtype)
    _call_on(dev, "hmoe_norm_modulate", x.data_ptr(), ldx, L._DT[x.dtype], L.ptr(weight), _dt0(weight), L.ptr(scale),
             L.ptr(shift), _dt0(shift if scale is None else scale), L.ptr(starts), B, T, d, float(eps), h.data_ptr(),
             L._DT[dtype])
    return h


def norm_modulate_bwd(dh, x, weight=None, scale=None, shift=None, starts=None, eps=1e-6, dres=None, dres_scale=1.0,
                      want=("weight", "scale", "shift")):
    """(dx, dweight, dscale, dshift) of norm_modulate, None for parameters that are absent or not in `want`; dres (T, d) of
    x's type, the gradient of x past the block, joins dx as dres_scale * dres.  dx has x's type, the others their
    parameters'."""
    T, d, ldx = _rows(x, "x")
    dev = x.device
    _on(dh, "dh", dev, (T, d), (_block_dtype(x.dtype, dh.dtype),))
    _on(weight, "weight", dev, (d,), _FLOATS)
    _on(dres, "dres", dev, (T, d), (x.dtype,))
    B = _sample_params(T, d, dev, starts, scale, "scale", shift, "shift")
    if scale is not None and shift is not None and scale.dtype != shift.dtype:
        raise TypeError(f"scale and shift must have one type (got {scale.dtype}, {shift.dtype})")
    dx = torch.empty(T, d, device=dev, dtype=x.dtype)
    dw = torch.empty_like(weight) if weight is not None and "weight" in want else None
    dsc = torch.empty_like(scale) if scale is not None and "scale" in want else None
    dsh = torch.empty_like(shift) if shift is not None and "shift" in want else None
    ws, ws_bytes = None, 0
    if dw is not None or dsc is not None or dsh is not None:
        ws_bytes = L.lib().hmoe_norm_modulate_bwd_workspace_size(T, d, B)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _call_on(dev, "hmoe_norm_modulate_bwd", dh.data_ptr(), L._DT[dh.dtype], x.data_ptr(), ldx, L._DT[x.dtype],
             L.ptr(weight), _dt0(weight), L.ptr(scale), L.ptr(shift), _dt0(shift if scale is None else scale),
             L.ptr(starts), B, T, d, float(eps), L.ptr(dres), float(dres_scale), dx.data_ptr(), L.ptr(dw), L.ptr(dsc),
             L.ptr(dsh), L.ptr(ws), ws_bytes)
    return dx, dw, dsc, dsh


def _slots(y, k, T, d, dev, inv_pos, add):
    if k < 1:
        raise ValueError(f"k = {k} slots")
    _on(y, "y", dev, (T * k, d), _FLOATS)
    _on(inv_pos, "inv_pos", dev, (T * k,), _I32)
    _on(add, "add", dev, (T, d), (y.dtype,))


def norm_residual(y, x, gate=None, weight=None, norm=True, starts=None, eps=1e-6, alpha=1.0, k=1, inv_pos=None, add=None):
    """out (T, d) = alpha * x + gate_b * weight * n, n = s / sqrt(mean(s^2) + eps) (s itself without norm): the gated
    residual behind a block.  s is the sum over the k slots of y (T*k, d) (plus add (T, d), the shared expert's output), what
    combine gives without its rounding; with inv_pos from the dispatch, slots routed nowhere add nothing.  gate (B, d) per
    sample as in norm_modulate, or (d,); padding rows get alpha * x.  out has the type of the stream x.  (The block's output
    comes first here; the differentiable norm_residual of the package takes the stream first.)"""
    T, d, ldx = _rows(x, "x")
    dev = x.device
    _block_dtype(x.dtype, y.dtype)
    _slots(y, k, T, d, dev, inv_pos, add)
    _on(weight, "weight", dev, (d,), _FLOATS)
    B = _sample_params(T, d, dev, starts, gate, "gate")
    out = torch.empty(T, d, device=dev, dtype=x.dtype)
    _call_on(dev, "hmoe_norm_residual", y.data_ptr(), L.ptr(inv_pos), k, L.ptr(add), L._DT[y.dtype], x.data_ptr(), ldx,
             L._DT[x.dtype], L.ptr(weight), _dt0(weight), L.ptr(gate), _dt0(gate), L.ptr(starts), B, T, d, int(bool(norm)),
             float(eps), float(alpha), out.data_ptr())
    return out


def norm_residual_bwd(dout, y, gate=None, weight=None, norm=True, starts=None, eps=1e-6, k=1, inv_pos=None, add=None,
                      want=("weight", "gate")):
    """(dy, dgate, dweight) of norm_residual, None for parameters that are absent or not in `want`: dy (T, d) of y's type is
    the gradient of the slots' sum (of every slot and of add); x's is alpha * dout."""
    _, d, ld = _rows(dout, "dout")
    T = dout.shape[0]
    dev = dout.device
    _on(dout, "dout", dev, (T, d), _FLOATS)
    _block_dtype(dout.dtype, y.dtype)
    _slots(y, k, T, d, dev, inv_pos, add)
    _on(weight, "weight", dev, (d,), _FLOATS)
    B = _sample_params(T, d, dev, starts, gate, "gate")
    dy = torch.empty(T, d, device=dev, dtype=y.dtype)
    dw = torch.empty_like(weight) if weight is not None and "weight" in want else None
    dg = torch.empty_like(gate) if gate is not None and "gate" in want else None
    ws, ws_bytes = None, 0
    if dw is not None or dg is not None:
        ws_bytes = L.lib().hmoe_norm_residual_bwd_workspace_size(T, d, B)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _call_on(dev, "hmoe_norm_residual_bwd", dout.data_ptr(), L._DT[dout.dtype], y.data_ptr(), L.ptr(inv_pos), k,
             L.ptr(add), L._DT[y.dtype], L.ptr(weight), _dt0(weight), L.ptr(gate), _dt0(gate), L.ptr(starts), B, T, d,
             int(bool(norm)), float(eps), dy.data_ptr(), L.ptr(dw), L.ptr(dg), L.ptr(ws), ws_bytes)
    return dy, dg, dw


def _dense(t):
    """Whether t's elements fill one stretch of memory (contiguous in some order of its dimensions)."""
    return t.is_contiguous() or t.permute(sorted(range(t.dim()), key=t.stride, reverse=True)).is_contiguous()


class GradList:
    """The tensors of a clipping call as the C entry points take them: addresses, element counts and types.  A program whose
    gradients stay in place (flat buckets, zero_grad(set_to_none=False)) may keep one from step to step."""

    def __init__(self, grads, out=None):
        grads = list(grads)
        self.n = len(grads)
        self.device = self._check(grads, "gradient")
        self.ptr = self._ptrs(grads)
        self.numel = array("q", list(map(torch.Tensor.numel, grads)))
        self.dt = self._types(grads)
        if out is None:
            out = grads
            self.out, self.odt = self.ptr, self.dt
        else:
            out = list(out)
            if len(out) != self.n:
                raise ValueError(f"{len(out)} outputs for {self.n} gradients")
            if self._check(out, "output") != self.device:
                raise ValueError("the gradients and outputs of a call live on one device")
            for g, o in zip(grads, out):
                if o is not g and (o.shape != g.shape or (o.stride() != g.stride() and g.numel() > 1)
                                   or o.dtype not in (g.dtype, torch.float32)):
                    raise ValueError("an output has its gradient's shape and strides, and its type or fp32")
            self.out, self.odt = self._ptrs(out), self._types(out)
            if not set(self.out).isdisjoint(self.ptr):  # (tensors without elements may share the address 0)
                held = {p for p, n in zip(self.ptr, self.numel) if n}
                if any(o != p and n and o in held for p, o, n in zip(self.ptr, self.out, self.numel)):
                    raise ValueError("an output lies over another gradient")
        self.keep = (grads, out)
        if len(set(self.out)) != self.n:
            used = [p for p, n in zip(self.out, self.numel) if n]
            if len(set(used)) != len(used):
                raise ValueError("a tensor is listed twice")

    # one pass per property, mapped over the tensors by the descriptor itself: a program clips hundreds of them, and the time
    # of this is the host's
    @staticmethod
    def _check(ts, name):
        devs = set(map(torch.Tensor.get_device, ts))
        if len(devs) > 1:
            raise ValueError(f"the {name}s of a call live on one device (got {sorted({str(t.device) for t in ts})})")
        dev = ts[0].device if ts else None
        if dev is not None and dev.type != "cuda":
            raise RuntimeError(f"a {name} must be a ROCm GPU tensor: the hmoe kernels have no CPU path")
        if not all(map(torch.Tensor.is_contiguous, ts)) and not all(map(_dense, ts)):
            raise ValueError(f"a {name}'s elements must be contiguous")
        return dev

    @staticmethod
    def _ptrs(ts):
        return array("Q", list(map(torch.Tensor.data_ptr, ts)))

    @staticmethod
    def _types(ts):
        kinds = list(map(torch.Tensor.dtype.__get__, ts))
        found = set(kinds)
        if not found.issubset(_FLOATS):
            raise TypeError(f"gradients and outputs are bf16, fp16 or fp32 (got {found})")
        if len(found) == 1:
            return array("i", [L._DT[kinds[0]]]) * len(kinds)
        return array("i", [L._DT[k] for k in kinds])


def _addr(a):
    return a.buffer_info()[0] if len(a) else None


def grad_sq_norm(grads):
    """(1,) fp64 on the device: the sum of the squares of every element of a list of gradients (or a GradList).  The order of the
    sum, and so its last bits, goes by the list and its tensors' addresses."""
    gl = grads if isinstance(grads, GradList) else GradList(grads)
    dev = gl.device if gl.device is not None else torch.device("cuda", torch.cuda.current_device())
    sq = torch.empty(1, device=dev, dtype=torch.float64)
    ws_bytes = L.lib().hmoe_grad_sq_norm_workspace_size(gl.n)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _call_on(dev, "hmoe_grad_sq_norm", _addr(gl.ptr), _addr(gl.numel), _addr(gl.dt), gl.n, sq.data_ptr(), ws.data_ptr(),
             ws_bytes)
    return sq


def grad_clip(grads, sq_norm, max_norm, out=None):
    """Scales a list of gradients (or a GradList) by min(1, max_norm / (norm + 1e-6)), norm = sqrt(sq_norm) -- in place, or
    into `out` (tensors of the gradients' shapes, of their types or fp32; a GradList has its own).  Outputs that overlap each
    other, another gradient or their own in another type are refused.  Returns the norm, () fp32 on the device."""
    if out is not None and isinstance(grads, GradList):
        raise ValueError("a GradList holds its outputs already: pass them to GradList")
    gl = grads if isinstance(grads, GradList) else GradList(grads, out)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm = {max_norm}")
    dev = sq_norm.device
    _on(sq_norm, "sq_norm", dev if gl.device is None else gl.device, (1,), (torch.float64,))
    L.require_gpu(sq_norm, "sq_norm")
    norm = torch.empty((), device=dev, dtype=torch.float32)
    try:
        _call_on(dev, "hmoe_grad_clip_f64", _addr(gl.ptr), _addr(gl.out), _addr(gl.numel), _addr(gl.dt), _addr(gl.odt),
                 gl.n, sq_norm.data_ptr(), max_norm, norm.data_ptr())
    except L.HmoeError as e:
        if e.code != L.ERR_OVERLAP:
            raise
        raise ValueError("a tensor to be written lies over another gradient or output of the call, or over its own gradient "
                         "in another type") from e
    return norm


# ---------------------------------------------------------------------------------------------------------------
# Experts in 8-bit floating point (e4m3 values, a power-of-two scale per block of 128)
# ---------------------------------------------------------------------------------------------------------------
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _f8_ld(K):
    return -(-K // 2048) * 16  # hmoe_f8_scale_ld: one byte per 128 columns, in whole 16 bytes


def quant_rows(x):
    """Rows x (M, K) bf16, fp16 or fp32 in 8 bits with a scale per 128 columns -> (q (M, K) float8_e4m3fn, s
    (M, ceil(K / 128)) float8_e8m0fnu): x is about q * s.  s is 2^e with the least e >= -126 that brings the block's largest finite
    value to at most 448; infinities and NaNs become NaN.  K a multiple of 16."""
    M, K, ld = _rows(x, "x")
    if K % 16:
        raise ValueError(f"x: width {K} must be a multiple of 16")
    q = torch.empty(M, K, device=x.device, dtype=_E4M3)
    s = torch.empty(M, _f8_ld(K), device=x.device, dtype=_E8M0)
    _call_on(x.device, "hmoe_f8_quant_rows", L.ptr(x), ld, L.dt(x), M, K, L.ptr(q), K, L.ptr(s), s.shape[1])
    return q, s[:, :-(-K // 128)]


def _f8_rows(q, s, block=128):
    """(M, K, row stride, scale row stride) of quantised rows."""
    L.require_gpu(q, "q")
    if q.dim() != 2 or q.dtype != _E4M3 or s.dtype != _E8M0:
        raise TypeError(f"quantised rows are (M, K) float8_e4m3fn with float8_e8m0fnu scales (got {q.dtype}, {s.dtype})")
    M, K = q.shape
    if s.device != q.device:
        raise ValueError(f"the scales are on {s.device}, the rows on {q.device}")
    if tuple(s.shape) != (M, -(-K // block)):
        raise ValueError(f"scales of shape {tuple(s.shape)}, expected {(M, -(-K // block))}")
    ld = q.stride(0) if M > 1 else K
    lds = s.stride(0) if M > 1 else max(s.stride(0), _f8_ld(K) if block == 128 else s.shape[1])
    if (K and q.stride(1) != 1) or ld < K or (s.shape[1] > 1 and s.stride(1) != 1):
        raise ValueError("quantised rows and their scales must be contiguous in themselves")
    if block == 128 and (ld % 16 or lds % 16 or lds < _f8_ld(K) or q.data_ptr() % 16 or s.data_ptr() % 16):
        raise ValueError("quantised rows and scale rows lie 16-byte aligned, as quant_rows gives them")
    return M, K, ld, lds


def dequant_rows(q, s, dtype=torch.float32, block=128):
    """The values of quantised rows (quant_rows; block=32: swiglu_pack's) -> (M, K) of `dtype` (fp32 holds them exactly, but
    for a number of more than 3.29e38, which may have been rounded up to 2^128)."""
    M, K, ld, lds = _f8_rows(q, s, block)
    if dtype not in _FLOATS:
        raise TypeError(f"dtype {dtype} not in {_FLOATS}")
    x = torch.empty(M, K, device=q.device, dtype=dtype)
    if K:
        _call_on(q.device, "hmoe_f8_dequant_rows", L.ptr(q), ld, L.ptr(s), lds, M, K, block, L.ptr(x), K, L.dt(dtype))
    return x


@dataclass
class F8Stack:
    """Expert weights (E, K, N) in 8 bits, laid out for the products: q (E, N, K) float8_e4m3fn with its scales s, and, for the
    gradient of the rows, grad_q (E, K, N) and grad_s.  halves = 2 for [gate | up] stacks (each half's blocks from its own first
    column).  Frozen: no gradient reaches the weights."""

    q: torch.Tensor
    s: torch.Tensor
    halves: int = 1
    grad_q: torch.Tensor | None = None
    grad_s: torch.Tensor | None = None

    @property
    def shape(self):
        """(E, K, N), as of the stack it was made from."""
        return torch.Size((self.q.shape[0], self.q.shape[2], self.q.shape[1]))

    @property
    def device(self):
        return self.q.device

    @classmethod
    def from_weights(cls, w, halves=1, grad=False):
        """w (E, K, N) bf16, fp16 or fp32, N contiguous; K and N / halves multiples of 16.  grad=True also keeps the layout that
        the gradient of the rows reads (as many bytes again)."""
        L.require_gpu(w, "w")
        if w.dim() != 3 or w.dtype not in _FLOATS:
            raise TypeError(f"w must be an (E, K, N) stack of bf16, fp16 or fp32 (got {tuple(w.shape)} {w.dtype})")
        E, K, N = w.shape
        if halves not in (1, 2) or min(E, K, N) < 1 or N % halves:
            raise ValueError(f"w {tuple(w.shape)} in {halves} halves")
        if K % 16 or N // halves % 16:
            raise ValueError(f"w {tuple(w.shape)}: K and N / halves must be multiples of 16")
        w = w.detach()
        if w.stride(2) != 1 or w.stride(1) < N or w.stride(1) % 8 or w.stride(0) % 8 or w.data_ptr() % 16:
            w = w.contiguous() if not w.is_contiguous() else w.clone()
        nb = -(-(N // halves) // 128)
        st = cls(torch.empty(E, N, K, device=w.device, dtype=_E4M3),
                 torch.zeros(E, halves * nb, _f8_ld(K), device=w.device, dtype=torch.uint8).view(_E8M0), halves)
        args = (L.ptr(w), L.dt(w), E, K, N, w.stride(0), w.stride(1))
        _call_on(w.device, "hmoe_f8_quant_stack", *args, halves, 1, L.ptr(st.q), L.ptr(st.s))
        if grad:
            st.grad_q = torch.empty(E, K, N, device=w.device, dtype=_E4M3)
            st.grad_s = torch.zeros(E, -(-K // 128), _f8_ld(N), device=w.device, dtype=torch.uint8).view(_E8M0)
            _call_on(w.device, "hmoe_f8_quant_stack", *args, 1, 0, L.ptr(st.grad_q), L.ptr(st.grad_s))
        return st

    def to(self, device):
        """The stack on another device."""
        return F8Stack(*(t.to(device) if isinstance(t, torch.Tensor) else t
                         for t in (self.q, self.s, self.halves, self.grad_q, self.grad_s)))

    def dequant(self):
        """The values it stands for, (E, K, N) fp32."""
        E, K, N = self.shape
        s = self.s.to(torch.float32)[:, :, :-(-K // 128)]
        rows = torch.cat([torch.arange(N // self.halves, device=s.device) // 128 + i * (s.shape[1] // self.halves)
                          for i in range(self.halves)])
        return (self.q.to(torch.float32) * s[:, rows].repeat_interleave(128, 2)[:, :, :K]).transpose(1, 2).contiguous()


def _f8_stack(w, name, dev, shape=None, halves=None):
    """Checks a stack handed to a C entry point (its fields are public)."""
    if not isinstance(w, F8Stack):
        raise TypeError(f"{name}: an F8Stack expected (got {type(w).__name__})")
    E, K, N = w.shape
    if shape is not None and any(want is not None and got != want for got, want in zip((E, K, N), shape)):
        raise ValueError(f"{name}: shape {(E, K, N)} does not match {shape}")
    if halves is not None and w.halves != halves:
        raise ValueError(f"{name}: a stack of {w.halves} halves, {halves} expected")
    _on(w.q, name, dev, (E, N, K), (_E4M3,))
    _on(w.s, name + " scales", dev, (E, w.halves * -(-(N // w.halves) // 128), _f8_ld(K)), (_E8M0,))
    return E, K, N


def _f8_idx(counts, a_idx, y_idx, scale, dev, E, M, rows, ld):
    """The checks that the grouped products share -> (counts, scale)."""
    counts = _on(counts if counts.dtype in (torch.int32, torch.int64) else counts.to(torch.int64), "counts", dev, (E,),
                 (torch.int32, torch.int64))
    if a_idx is not None:
        _on(a_idx, "a_idx", dev, (M,), _I32)
        if rows * ld >= 2 ** 31 - 32768:
            raise ValueError("a gathered through a_idx must span less than 2 GiB (32-bit row offsets)")
    if rows < (min(1, M) if a_idx is not None else M):
        raise ValueError(f"a: {rows} rows for {M} of the product")
    _on(y_idx, "y_idx", dev, (M,), _I32)
    if scale is not None:
        scale = _on(scale if scale.dtype in _FLOATS else scale.float(), "scale", dev, (M,), _FLOATS)
    return counts, scale


def quant_mm_f8(x, w, counts, M=None, a_idx=None, y_idx=None, scale=None, dtype=None):
    """grouped_mm_f8 of x's rows quantised on the way (quant_rows), in one call: x (rows, K) bf16, fp16 or fp32 -> (M, N) of
    `dtype`, x's type by default."""
    E, K, N = _f8_stack(w, "w", x.device)
    return _quant_mm(x, w.q, w.s, E, K, N, w.halves, counts, M, a_idx, y_idx, scale, dtype)


def _quant_mm(x, wq, ws, E, K, N, halves, counts, M, a_idx, y_idx, scale, dtype):
    rows, K_, ld = _rows(x, "x")
    if K_ != K:
        raise ValueError(f"x has {K_} columns, the stack {K} rows")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise TypeError(f"dtype {dtype} not in {_FLOATS}")
    dev = x.device
    M = (a_idx.numel() if a_idx is not None else rows) if M is None else M
    counts, scale = _f8_idx(counts, a_idx, y_idx, scale, dev, E, M, rows, K)
    n = rows * (K + _f8_ld(K)) + 16
    tmp = torch.empty(n, device=dev, dtype=torch.uint8)
    y = torch.empty(M, N, device=dev, dtype=dtype)
    _call_on(dev, "hmoe_f8_quant_mm", x.data_ptr(), ld, L.dt(x), rows, wq.data_ptr(), ws.data_ptr(), E, K, N, halves,
             counts.data_ptr(), L.dt(counts), M, L.ptr(a_idx), L.ptr(y_idx), L.ptr(scale),
             L.dt(scale) if scale is not None else 0, 0, y.data_ptr(), N, L.dt(dtype), tmp.data_ptr(), n)
    return y


def _f8_mm(q, s, wq, ws, E, K, N, halves, counts, M, a_idx, y_idx, scale, dtype, scale_by_y=False):
    """hmoe_f8_grouped_mm on checked stacks."""
    rows, K_, ld, lds = _f8_rows(q, s)
    dev = q.device
    if K_ != K:
        raise ValueError(f"a has {K_} columns, the stack {K} rows")
    if dtype not in _FLOATS:
        raise TypeError(f"dtype {dtype} not in {_FLOATS}")
    counts, scale = _f8_idx(counts, a_idx, y_idx, scale, dev, E, M, rows, ld)
    y = torch.empty(M, N, device=dev, dtype=dtype)
    _call_on(dev, "hmoe_f8_grouped_mm", L.ptr(q), ld, L.ptr(s), lds, rows, L.ptr(wq), L.ptr(ws), E, K, N, halves, L.ptr(counts),
             L.dt(counts), M, L.ptr(a_idx), L.ptr(y_idx), L.ptr(scale), L.dt(scale) if scale is not None else 0,
             int(scale_by_y), L.ptr(y), N, L.dt(dtype))
    return y


def grouped_mm_f8(q, s, w, counts, M=None, a_idx=None, y_idx=None, scale=None, dtype=torch.bfloat16):
    """grouped_mm on rows in 8 bits (quant_rows) and an F8Stack: y[y_idx[r] or r] = scale[r] * a[a_idx[r] or r] @ w[e(r)] ->
    (M, N) of `dtype` (bf16, fp16 or fp32), rounded once.  The 8-bit matrix instructions drop what lies below 2^-13 of the largest of
    eight consecutive k's products and add the rest in fp32: some 2^-16 of a sum, which 16-bit outputs do not show; of fp32 outputs
    about 16 bits hold.  Index values are trusted, as in grouped_mm.  Rows
    that counts name for no expert are zeros; with y_idx they are not written."""
    E, K, N = _f8_stack(w, "w", q.device)
    M = (a_idx.numel() if a_idx is not None else q.shape[0]) if M is None else M
    return _f8_mm(q, s, w.q, w.s, E, K, N, w.halves, counts, M, a_idx, y_idx, scale, dtype)


def grouped_mm_f8_bwd(dy, w, counts):
    """The gradient of grouped_mm_f8's rows: dy (M, N) bf16, fp16 or fp32, sorted by expert, is quantised along N and multiplied
    by the stack's other layout (F8Stack.from_weights(..., grad=True)) -> (M, K) of dy's type."""
    E, K, N = _f8_stack(w, "w", dy.device)
    if w.grad_q is None:
        raise ValueError("this F8Stack was made without grad=True: it has no layout for the gradient of the rows")
    _on(w.grad_q, "w.grad_q", dy.device, (E, K, N), (_E4M3,))
    _on(w.grad_s, "w.grad_s", dy.device, (E, -(-K // 128), _f8_ld(N)), (_E8M0,))
    return _quant_mm(dy, w.grad_q, w.grad_s, E, N, K, 1, counts, None, None, None, None, None)


def gate_up_swiglu_f8(q, s, wgu, counts, M=None, a_idx=None, wide=False):
    """act = silu(g) * u of [g | u] = a[a_idx] @ wgu[e] in fp32, in 8 bits -> (act (M, h) float8_e4m3fn, its scales
    (M, ceil(h / 128)) float8_e8m0fnu), ready for grouped_mm_f8 with the down stack.  wgu: an F8Stack (E, d, 2h) of 2 halves.
    wide: the products on the bf16 matrix instructions, exact but for the fp32 sums, at half the rate (the 8-bit ones drop some
    2^-16 of a sum, which moves about one act in a thousand across a border of its 8 bits); moe_experts takes it for fp16."""
    E, d, h2 = _f8_stack(wgu, "wgu", q.device, halves=2)
    rows, K, ld, lds = _f8_rows(q, s)
    dev, h = q.device, h2 // 2
    M = (a_idx.numel() if a_idx is not None else rows) if M is None else M
    if K != d:
        raise ValueError(f"a has {K} columns, wgu {d} rows")
    counts, _ = _f8_idx(counts, a_idx, None, None, dev, E, M, rows, ld)
    act = torch.empty(M, h, device=dev, dtype=_E4M3)
    act_s = torch.empty(M, _f8_ld(h), device=dev, dtype=_E8M0)
    _call_on(dev, "hmoe_f8_gate_up_swiglu", L.ptr(q), ld, L.ptr(s), lds, rows, L.ptr(a_idx), L.ptr(wgu.q), L.ptr(wgu.s), E, d, h,
             L.ptr(counts), L.dt(counts), M, int(bool(wide)), L.ptr(act), L.ptr(act_s))
    return act, act_s[:, :-(-h // 128)]


def _moe_experts_f8(x, ids, tw, wgu, wd):
    """moe_experts over F8Stacks (hmoe_f8_moe_experts)."""
    T, k = ids.shape
    if x.dim() != 2 or x.shape[0] != T or x.stride(1) != 1:
        raise ValueError(f"x must be a ({T}, d) matrix with contiguous rows (got {tuple(x.shape)})")
    L.require_gpu(x, "x")
    dt, d, dev = _act_dtype(x, "x"), x.shape[1], x.device
    E, _, h2 = _f8_stack(wgu, "wgu", dev, (None, d, None), 2)
    h = h2 // 2
    _f8_stack(wd, "wd", dev, (E, h, d), 1)
    _on(ids, "topk_ids", dev, (T, k), (torch.int32, torch.int64))
    tw = _on(tw if tw.dtype in _FLOATS else tw.float(), "topk_weight", dev, (T, k), _FLOATS)
    ws_bytes = L.lib().hmoe_f8_moe_experts_workspace_size(T, d, E, k, h)
    if ws_bytes == 0:
        raise ValueError(f"moe_experts: unsupported sizes T={T} d={d} E={E} k={k} h={h}")
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    y = torch.empty(T * k, d, device=dev, dtype=x.dtype)
    inv = torch.empty(T * k, device=dev, dtype=torch.int32)
    n_invalid = torch.empty(1, device=dev, dtype=torch.int32)
    _call_on(dev, "hmoe_f8_moe_experts", L.ptr(x), x.stride(0) if T > 1 else d, dt, L.ptr(ids), L.dt(ids), L.ptr(tw), L.dt(tw),
             L.ptr(wgu.q), L.ptr(wgu.s), L.ptr(wd.q), L.ptr(wd.s), T, d, E, k, h, L.ptr(y), L.ptr(inv), L.ptr(n_invalid),
             L.ptr(ws), ws_bytes)
    return y, inv, n_invalid


# ---------------------------------------------------------------------------------------------------------------
# SwiGLU with an 8-bit checkpoint
# ---------------------------------------------------------------------------------------------------------------
@dataclass
class PackedGU:
    """[g | u] (M, 2h) in 8 bits: q (M, 2h) float8_e4m3fn, s (M, 2 ceil(h / 32)) float8_e8m0fnu, a scale per 32 columns of g, then
    of u; dtype: the type it had."""

    q: torch.Tensor
    s: torch.Tensor
    dtype: torch.dtype

    def dequant(self, dtype=torch.float32):
        """The values kept, (M, 2h)."""
        h, nb = self.q.shape[1] // 2, self.s.shape[1] // 2
        return torch.cat([dequant_rows(self.q[:, i * h:(i + 1) * h], self.s[:, i * nb:(i + 1) * nb], dtype, block=32)
                          for i in range(2)], 1)


def swiglu_pack(gu):
    """gu (M, 2h) = [g | u] bf16 or fp16 -> (act (M, h) = silu(g) * u, rounded once; PackedGU, g and u in 8 bits).  h a multiple
    of 8; infinities and NaNs are kept as NaN."""
    M, h2, ld = _rows(gu, "gu", _H16)
    if h2 % 16:
        raise ValueError(f"gu: width {h2} must be twice a multiple of 8")
    h, dev = h2 // 2, gu.device
    act = torch.empty(M, h, device=dev, dtype=gu.dtype)
    kept = PackedGU(torch.empty(M, h2, device=dev, dtype=_E4M3), torch.empty(M, 2 * -(-h // 32), device=dev, dtype=_E8M0), gu.dtype)
    _call_on(dev, "hmoe_swiglu_pack", L.ptr(gu), ld, M, h, L.ptr(act), L.ptr(kept.q), L.ptr(kept.s), L.dt(gu))
    return act, kept


def swiglu_pack_bwd(dh, kept, w=None, order=None, want_act=True, want_dw=True):
    """The backward of swiglu_pack from what it kept -> (dgu (M, 2h), act (M, h) or None, dw (M,) fp32 or None).  dh (M, h) of
    gu's type; w (M,) multiplies its rows (the routing weight); act is the activation of the kept values and dw[order[r] or r]
    = <dh[r], act[r]>, w's gradient (rows of order -1 have none, places of dw that order does not name are 0)."""
    M, h, ld = _rows(dh, "dh", _H16)
    dev = dh.device
    if ld != h:
        dh = dh.contiguous()
    if dh.dtype != kept.dtype:
        raise TypeError(f"dh: dtype {dh.dtype}, the checkpoint is of {kept.dtype}")
    _on(kept.q, "the checkpoint", dev, (M, 2 * h), (_E4M3,))
    _on(kept.s, "the checkpoint's scales", dev, (M, 2 * -(-h // 32)), (_E8M0,))
    w = _on(w, "w", dev, (M,), _FLOATS)
    order = _on(order, "order", dev, (M,), _I32)
    dgu = torch.empty(M, 2 * h, device=dev, dtype=dh.dtype)
    act = torch.empty(M, h, device=dev, dtype=dh.dtype) if want_act else None
    dw = (torch.empty if order is None else torch.zeros)(M, device=dev, dtype=torch.float32) if want_dw else None
    _call_on(dev, "hmoe_swiglu_pack_bwd", L.ptr(dh), L.ptr(kept.q), L.ptr(kept.s), L.ptr(w), L.dt(w) if w is not None else 0, M, h,
             L.ptr(dgu), L.ptr(act), L.ptr(order), L.ptr(dw), L.dt(dh))
    return dgu, act, dw


# ---------------------------------------------------------------------------------------------------------------
# A routed layer for a few tokens
# ---------------------------------------------------------------------------------------------------------------
FEW_TOKENS = 16  # the most a call takes


def _few_args(x, k, wgu, wd, wgu_s, wd_s, add):
    """Checks of few_experts and few_forward -> (T, d, row stride, E, h, weight pointers and types, workspace, out)."""
    if x.dim() != 2 or not x.is_cuda:
        L.require_gpu(x, "x")
        raise ValueError(f"x must be a (T, d) matrix (got {tuple(x.shape)})")
    dt, dev = _act_dtype(x, "x"), x.device
    T, d = x.shape
    if T > FEW_TOKENS or not 1 <= k <= 16:
        raise ValueError(f"{T} tokens in {k} slots: at most {FEW_TOKENS} in 1 to 16")
    ld = x.stride(0) if T > 1 else d
    if T and (x.stride(1) != 1 or ld < d or ld % 8 or x.data_ptr() % 16):
        raise ValueError(f"x: rows must be contiguous, 16-byte aligned, with a row stride of a multiple of 8 (strides {x.stride()})")
    if isinstance(wgu, F8Stack) or isinstance(wd, F8Stack):
        if wgu_s is not None or wd_s is not None:
            raise ValueError("F8Stacks hold their own scales")
        E, _, h2 = _f8_stack(wgu, "wgu", dev, (None, d, None), 2)
        h = h2 // 2
        _f8_stack(wd, "wd", dev, (E, h, d), 1)
        w_dt = L.DT_F8
        ws = (L.ptr(wgu.q), L.ptr(wgu.s), 0, L.ptr(wd.q), L.ptr(wd.s), 0, w_dt)
    else:
        if wgu.dim() != 3 or wd.dim() != 3 or wgu.dtype not in (x.dtype, torch.int8) or wd.dtype != wgu.dtype:
            raise TypeError(f"wgu (E, d, 2h) and wd (E, h, d) of x's type, int8 or F8Stacks expected (got {wgu.dtype}, {wd.dtype})")
        E, h = wgu.shape[0], wd.shape[1]
        _on(wgu, "wgu", dev, (E, d, 2 * h), (wgu.dtype,))
        _on(wd, "wd", dev, (E, h, d), (wd.dtype,))
        wgu_s, wd_s = _w_scale(wgu, wgu_s, 2 * h), _w_scale(wd, wd_s, d)
        for t, name in ((wgu_s, "wgu_s"), (wd_s, "wd_s")):
            if t is not None:
                _on(t, name, dev, t.shape, (t.dtype,))
        w_dt = L.dt(wgu)
        ws = (L.ptr(wgu), L.ptr(wgu_s), L.dt(wgu_s) if wgu_s is not None else 0, L.ptr(wd), L.ptr(wd_s),
              L.dt(wd_s) if wd_s is not None else 0, w_dt)
    _on(add, "add", dev, (T, d), (x.dtype,))
    n = L.lib().hmoe_few_workspace_size(T, d, E, k, h, w_dt, dt)
    if n == 0 and T:
        raise ValueError(f"few tokens: unsupported sizes T={T} d={d} E={E} k={k} h={h}")
    return T, d, ld, E, h, ws, torch.empty(n, device=dev, dtype=torch.uint8), torch.empty(T, d, device=dev, dtype=x.dtype)


def few_experts(x, ids, tw, wgu, wd, wgu_s=None, wd_s=None, add=None, want_invalid=False):
    """The experts of a routed layer and the sum over its slots for up to 16 tokens, in two kernels (hmoe_few_experts): moe_experts
    and combine with fp32 sums throughout, rounded once (the activation enters its product with 16 significant bits, past bf16's
    largest number as an infinity) -> out (T, d).  x (T, d) bf16 or fp16; ids (T, k) int32 / int64, those outside
    [0, E) add nothing; tw (T, k); wgu (E, d, 2h) and wd (E, h, d) of x's type, int8 with scales, or F8Stacks; add (T, d) of x's
    type (a shared expert's output) joins the sum.  want_invalid: (out, n_invalid (1,) int32), how many ids named no expert."""
    T, k = ids.shape
    T_, d, ld, E, h, w, ws, out = _few_args(x, k, wgu, wd, wgu_s, wd_s, add)
    dev = x.device
    _on(ids, "topk_ids", dev, (T_, k), (torch.int32, torch.int64))
    tw = _on(tw if tw.dtype in _FLOATS else tw.float(), "topk_weight", dev, (T_, k), _FLOATS)
    bad = torch.zeros(1, device=dev, dtype=torch.int32) if want_invalid else None
    _call_on(dev, "hmoe_few_experts", L.ptr(x), ld, L.dt(x), L.ptr(ids), L.dt(ids), L.ptr(tw), L.dt(tw), *w, T, d, E, k, h,
             L.ptr(add), L.ptr(out), L.ptr(bad), L.ptr(ws), ws.numel())
    return (out, bad) if want_invalid else out


def few_forward(x, wr, wgu, wd, k, bias=None, renorm=True, scaling=1.0, add=None):
    """moe_forward for up to 16 tokens in two kernels (hmoe_few_forward), rounded as few_experts does -> (out (T, d),
    topk_ids (T, k) int32, topk_w (T, k) fp32: those of route_topk).  bf16; add (T, d) joins the sum."""
    _router_args(x, wr)
    T, d, ld, E, h, w, ws, out = _few_args(x, k, wgu, wd, None, None, add)
    dev = x.device
    if isinstance(wgu, F8Stack) or wgu.dtype != torch.bfloat16:
        raise TypeError("few_forward takes bf16 experts (few_experts any, with the routing given)")
    _on(wr, "router weight", dev, (E, d), _BF16)
    if not 1 <= k <= E:
        raise ValueError(f"top_k = {k} must lie in [1, {E}]")
    if bias is not None:
        bias = _on(bias.to(torch.float32), "logit bias", dev, (E,), (torch.float32,))
    ids = torch.empty(T, k, device=dev, dtype=torch.int32)
    tw = torch.empty(T, k, device=dev, dtype=torch.float32)
    _call_on(dev, "hmoe_few_forward", L.ptr(x), ld, L.ptr(wr), L.ptr(bias), w[0], w[3], T, d, E, k, h, int(bool(renorm)),
             float(scaling), L.ptr(add), L.ptr(out), L.ptr(ids), L.ptr(tw), L.ptr(ws), ws.numel())
    return out, ids, tw
