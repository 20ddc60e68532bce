"""torch-tensor wrappers over the libpmoe C ABI (one function per entry point).

Every function takes device tensors, checks dtype/shape/contiguity on the
host, and enqueues the HIP kernels on torch's current stream.  Packed
quantized words travel as ``torch.int32`` (same bits as the u32 of the
format); bf16 data as ``torch.bfloat16``.  There is no CPU path: without the
built library every call raises ``PmoeError``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import Geom, RouteCfg, check, lib

_WS: dict = {}
_MOE_WS: dict = {}
_WS_BYTES: dict = {}   # workspace bytes by the sizes that they depend on
# Workspaces handed out before a larger call replaced them.  They are never
# freed: a HIP graph captured over an earlier call keeps their raw pointers,
# and a replay must not write into memory torch has given to another tensor.
_RETIRED: dict = {"dispatch": [], "MoE": []}
# Pinned host words the workspaces' error words are copied into at sync points.
_ERR_HOST: dict = {}


def _ptr(t):
    """t's address as the binding's pointer arguments take it (building a
    ctypes object for it costs as much again)."""
    return None if t is None else t.data_ptr()


def _stream():
    """The current device's current stream.  Read as a raw handle: building
    torch's Stream object takes 4 us, and a paged decode layer asks six times."""
    if not torch.cuda.is_initialized():
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))


def _stream_of(t):
    """The current stream for work on t, which must be on the current device
    (launches go there)."""
    index = t.get_device()
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on {t.device}, but the current device is "
                         f"cuda:{torch._C._cuda_getDevice()}: call under torch.cuda.device")
    return torch._C._cuda_getCurrentRawStream(index)


def _fits(t, dtype, shape, index) -> bool:
    """Whether t is a contiguous tensor of that type and shape on GPU ``index``:
    the whole check of the usual call, a tenth of the time of the checks one by
    one that name what is wrong."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape
            and t.get_device() == index and t.is_contiguous())


def _same_device(a, b, name):
    if a.device != b.device:
        raise ValueError(f"{name}: on {b.device}, the other tensors on {a.device}")


def _need(t, dtype, name, ndim=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be a device tensor (got {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name}: expected {ndim} dims, got {tuple(t.shape)}")


def _grown(cache: dict, key, nbytes: int, device, what: str):
    """The cached buffer of at least nbytes, or a new one that replaces it
    (the old one is retired, not freed).  Growth is by at least 1.5x, so a
    sequence of larger calls retires only a few buffers.  Growing while the
    current stream is being captured into a graph raises: the capture would
    hold a pointer that a later, larger eager call cannot replace."""
    buf = cache.get(key)
    if buf is not None and buf.numel() >= nbytes:
        return buf, False
    if torch.cuda.is_current_stream_capturing():
        raise _lib.PmoeError(f"{what} workspace would grow to {nbytes} B during graph capture; "
                             "run the largest call once before capturing")
    size = max(int(nbytes), 256)
    if buf is not None:
        size = max(size, buf.numel() * 3 // 2)
        _RETIRED[what].append(buf)
    buf = torch.empty(size, dtype=torch.uint8, device=device)
    cache[key] = buf
    return buf, True


def workspace(nbytes: int, device) -> torch.Tensor:
    """A cached uint8 scratch tensor of at least nbytes on device."""
    return _grown(_WS, torch.device(device).index or 0, nbytes, device, "dispatch")[0]


# ---------------------------------------------------------------- routing

def router_logits(x: torch.Tensor, w: torch.Tensor, logit_bias=None) -> torch.Tensor:
    """fp32 logits [N, E] of x [N, D] bf16 against w [E, D] bf16."""
    _need(x, torch.bfloat16, "x", 2)
    _need(w, torch.bfloat16, "w", 2)
    n, d = x.shape
    e = w.shape[0]
    if w.shape[1] != d:
        raise ValueError("router weight hidden size mismatch")
    if logit_bias is not None:
        _need(logit_bias, torch.float32, "logit_bias", 1)
    out = torch.empty((n, e), dtype=torch.float32, device=x.device)
    check(lib().pmoe_router_logits(_ptr(x), _ptr(w), _ptr(logit_bias), n, d, e, _ptr(out),
                                   _stream()), "pmoe_router_logits")
    return out


def route_softmax_topk(logits: torch.Tensor, k: int, norm_topk_prob: bool = True):
    _need(logits, torch.float32, "logits", 2)
    n, e = logits.shape
    inds = torch.empty((n, k), dtype=torch.int32, device=logits.device)
    wts = torch.empty((n, k), dtype=torch.float32, device=logits.device)
    check(lib().pmoe_route_softmax_topk(_ptr(logits), n, e, k, int(bool(norm_topk_prob)),
                                        _ptr(inds), _ptr(wts), _stream()),
          "pmoe_route_softmax_topk")
    return inds, wts


def route_sigmoid_group_topk(logits, bias, n_group: int, topk_group: int, k: int,
                             norm_topk_prob: bool = True, routed_scale: float = 1.0):
    _need(logits, torch.float32, "logits", 2)
    _need(bias, torch.float32, "bias", 1)
    n, e = logits.shape
    inds = torch.empty((n, k), dtype=torch.int32, device=logits.device)
    wts = torch.empty((n, k), dtype=torch.float32, device=logits.device)
    check(lib().pmoe_route_sigmoid_group_topk(
        _ptr(logits), _ptr(bias), n, e, n_group, topk_group, k, int(bool(norm_topk_prob)),
        float(routed_scale), _ptr(inds), _ptr(wts), _stream()), "pmoe_route_sigmoid_group_topk")
    return inds, wts


# ---------------------------------------------------------------- dispatch

def dispatch(inds: torch.Tensor, n_experts: int) -> dict:
    """Stable grouping of the flat ids by expert (see pmoe_dispatch)."""
    _need(inds, torch.int32, "inds")
    rows = inds.numel()
    dev = inds.device
    out = {
        "order": torch.empty(rows, dtype=torch.int32, device=dev),
        "counts": torch.empty(n_experts, dtype=torch.int32, device=dev),
        "offsets": torch.empty(n_experts + 1, dtype=torch.int32, device=dev),
        "inv": torch.empty(rows, dtype=torch.int32, device=dev),
        "active": torch.empty(n_experts, dtype=torch.int32, device=dev),
        "n_active": torch.empty(1, dtype=torch.int32, device=dev),
    }
    wsb = lib().pmoe_dispatch_workspace(rows, n_experts)
    ws = workspace(wsb, dev)
    check(lib().pmoe_dispatch(_ptr(inds), rows, n_experts, _ptr(out["order"]),
                              _ptr(out["counts"]), _ptr(out["offsets"]), _ptr(out["inv"]),
                              _ptr(out["active"]), _ptr(out["n_active"]), _ptr(ws), ws.numel(),
                              _stream()), "pmoe_dispatch")
    return out


# ---------------------------------------------------------------- format

def quantize(w: torch.Tensor, bits: int, group: int = 64, out=None):
    """fp32 [R, C] -> (q int32 [R, C*bits/32], scales bf16, biases bf16).
    ``out`` = (q, s, b) contiguous tensors to write into (e.g. slab views)."""
    _need(w, torch.float32, "w", 2)
    r, c = w.shape
    if c % group or (c * bits) % 32:
        raise ValueError("columns must be a multiple of the group size")
    if out is None:
        q = torch.empty((r, c * bits // 32), dtype=torch.int32, device=w.device)
        s = torch.empty((r, c // group), dtype=torch.bfloat16, device=w.device)
        b = torch.empty((r, c // group), dtype=torch.bfloat16, device=w.device)
    else:
        q, s, b = out
        for t, dt, shape, name in ((q, torch.int32, (r, c * bits // 32), "q"),
                                   (s, torch.bfloat16, (r, c // group), "scales"),
                                   (b, torch.bfloat16, (r, c // group), "biases")):
            _need(t, dt, name)
            if tuple(t.shape) != shape:
                raise ValueError(f"{name}: expected {shape}, got {tuple(t.shape)}")
    check(lib().pmoe_quantize(_ptr(w), r, c, bits, group, _ptr(q), _ptr(s), _ptr(b), _stream()),
          "pmoe_quantize")
    return q, s, b


def dequant(q, scales, biases, bits: int, group: int = 64) -> torch.Tensor:
    _need(q, torch.int32, "q", 2)
    _need(scales, torch.bfloat16, "scales", 2)
    _need(biases, torch.bfloat16, "biases", 2)
    r = q.shape[0]
    c = q.shape[1] * 32 // bits
    out = torch.empty((r, c), dtype=torch.bfloat16, device=q.device)
    check(lib().pmoe_dequant(_ptr(q), _ptr(scales), _ptr(biases), r, c, bits, group, _ptr(out),
                             _stream()), "pmoe_dequant")
    return out


_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def mx4_quantize(w: torch.Tensor, out=None):
    """w [R, C] of fp32, bf16 or fp16 -> (q int32 [R, C/8], scales uint8
    [R, C/32]) in the microscaled 4-bit format (pmoe_mx4_quantize).  ``out`` =
    (q, scales) contiguous tensors to write into (e.g. slab views)."""
    if not isinstance(w, torch.Tensor) or w.dtype not in _DTYPES:
        raise TypeError("w: expected an fp32, bf16 or fp16 tensor")
    if not (w.dim() == 2 and w.is_cuda and w.is_contiguous()):
        _need(w, w.dtype, "w", 2)
    r, c = w.shape
    if c == 0 or c % 32:
        raise ValueError("columns must be a multiple of the group size, 32")
    if out is None:
        q = w.new_empty((r, c // 8), dtype=torch.int32)
        s = w.new_empty((r, c // 32), dtype=torch.uint8)
    else:
        q, s = out
        for t, dt, shape, name in ((q, torch.int32, (r, c // 8), "q"),
                                   (s, torch.uint8, (r, c // 32), "scales")):
            _need(t, dt, name)
            if tuple(t.shape) != shape:
                raise ValueError(f"{name}: expected {shape}, got {tuple(t.shape)}")
            _same_device(w, t, name)
    if r:
        check(lib().pmoe_mx4_quantize(w.data_ptr(), _DTYPES[w.dtype], r, c, q.data_ptr(),
                                      s.data_ptr(), _stream_of(w)), "pmoe_mx4_quantize")
    return q, s


def mx4_dequant(q: torch.Tensor, scales: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values [R, C] of microscaled 4-bit words q [R, C/8] and scales
    [R, C/32], rounded once to ``dtype`` (fp32, bf16 or fp16)."""
    _need(q, torch.int32, "q", 2)
    if dtype not in _DTYPES:
        raise TypeError("dtype: expected fp32, bf16 or fp16")
    r, c = q.shape[0], q.shape[1] * 8
    if not (c and c % 32 == 0 and _fits(scales, torch.uint8, (r, c // 32), q.get_device())):
        _need(scales, torch.uint8, "scales", 2)
        if c == 0 or c % 32 or tuple(scales.shape) != (r, c // 32):
            raise ValueError(f"scales: expected {(r, c // 32)} for words {tuple(q.shape)} of "
                             f"whole groups, got {tuple(scales.shape)}")
        _same_device(q, scales, "scales")
    out = q.new_empty((r, c), dtype=dtype)
    if r:
        check(lib().pmoe_mx4_dequant(q.data_ptr(), scales.data_ptr(), r, c, _DTYPES[dtype],
                                     out.data_ptr(), _stream_of(q)), "pmoe_mx4_dequant")
    return out


# ---------------------------------------------------------------- experts

def moe_workspace(g: Geom, n: int, k: int, shared: int, n_experts: int, device,
                  fresh: bool = False) -> torch.Tensor:
    """Workspace of the expert entry points (pmoe_moe_workspace bytes).  Its
    synchronisation header is zeroed on allocation (pmoe_moe_workspace_init);
    the cached buffer is separate from the dispatch scratch so nothing else
    ever writes the header.  fresh=True returns a new, private buffer."""
    sizes = (g.hidden, g.inter, g.group, n, k, shared, n_experts)
    nb = _WS_BYTES.get(sizes)
    if nb is None:
        nb = max(int(lib().pmoe_moe_workspace(ctypes.byref(g), n, k, shared, n_experts)), 256)
        if len(_WS_BYTES) >= 4096:
            _WS_BYTES.clear()
        _WS_BYTES[sizes] = nb
    if fresh:
        buf = torch.empty(nb, dtype=torch.uint8, device=device)
        check(lib().pmoe_moe_workspace_init(_ptr(buf), buf.numel(), _stream()),
              "pmoe_moe_workspace_init")
        return buf
    index = (device if isinstance(device, torch.device) else torch.device(device)).index or 0
    buf = _MOE_WS.get(index)
    if buf is not None and buf.numel() >= nb:
        return buf
    buf, new = _grown(_MOE_WS, index, nb, device, "MoE")
    if new:
        check(lib().pmoe_moe_workspace_init(_ptr(buf), buf.numel(), _stream()),
              "pmoe_moe_workspace_init")
    return buf


def _live_moe_workspaces():
    return list(_MOE_WS.values()) + _RETIRED["MoE"]


def note_workspace_errors() -> None:
    """Enqueue, on the current stream, copies of every cached MoE
    workspace's error word into pinned host memory (no wait).  A caller that
    synchronises the stream next reads them with ``raise_workspace_errors``."""
    for ws in _live_moe_workspaces():
        host = _ERR_HOST.get(ws.data_ptr())
        if host is None:
            host = _ERR_HOST[ws.data_ptr()] = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        check(lib().pmoe_moe_workspace_error_async(_ptr(ws), _ptr(host), _stream()),
              "pmoe_moe_workspace_error_async")


def raise_workspace_errors() -> None:
    """After a stream sync that followed ``note_workspace_errors``: raise
    PmoeError if a grid barrier of the one-launch decode timed out (those
    layer outputs are NaN).  The failed workspace is re-initialised first,
    so the next call runs normally."""
    words = {}
    for ws in _live_moe_workspaces():
        host = _ERR_HOST.get(ws.data_ptr())
        words[ws.data_ptr()] = 0 if host is None else host.item()
    bad = [ws for ws in _live_moe_workspaces() if words[ws.data_ptr()] != 0]
    if not bad:
        return
    err = 0
    for ws in bad:
        err |= words[ws.data_ptr()]
        _ERR_HOST[ws.data_ptr()].zero_()
        check(lib().pmoe_moe_workspace_init(_ptr(ws), ws.numel(), _stream()),
              "pmoe_moe_workspace_init")
    what = []
    if err & 1:
        what.append("a barrier wait timed out (a block was not resident in time)")
    if err & 2:
        what.append("the blocks of one group of the expert-per-XCD launch ran on "
                    "different XCDs")
    raise _lib.PmoeError("one-launch decode: " + "; ".join(what or [f"error word {err:#x}"])
                         + "; the affected layer outputs are NaN")


def check_workspace_errors() -> None:
    """Synchronising form of note + raise, for sync points of their own
    (get_stats)."""
    note_workspace_errors()
    torch.cuda.current_stream().synchronize()
    raise_workspace_errors()


def set_split_probe(on: bool) -> None:
    """Debug: make the expert-per-XCD decode's group 0 look split across two
    XCDs (pmoe_set_split_probe), so its placement check fires."""
    check(lib().pmoe_set_split_probe(int(bool(on))), "pmoe_set_split_probe")


def set_barrier_spin(ticks: int) -> None:
    """Debug: grid-barrier poll limit of later one-launch decode calls in
    100 MHz ticks (0 = the default 0.5 s); see pmoe_set_barrier_spin."""
    check(lib().pmoe_set_barrier_spin(int(ticks)), "pmoe_set_barrier_spin")


def workspace_error(ws: torch.Tensor) -> int:
    """The sticky error word of a MoE workspace header (synchronises)."""
    err = ctypes.c_uint32()
    check(lib().pmoe_moe_workspace_status(_ptr(ws), ctypes.byref(err), _stream()),
          "pmoe_moe_workspace_status")
    return int(err.value)


def _table_ptr(table, n_experts: int = 0):
    if isinstance(table, torch.Tensor):
        _need(table, torch.int32, "table", 1)
        if table.numel() < n_experts:
            raise ValueError(f"table holds {table.numel()} of {n_experts} experts")
        return table.data_ptr()
    return int(table)


def _rows_of(x, n, g, inds):
    """x is bf16 [n, hidden] beside inds: says what is not."""
    _need(x, torch.bfloat16, "x", 2)
    if x.shape != (n, g.hidden):
        raise ValueError(f"x must be [{n}, {g.hidden}], got {tuple(x.shape)}")
    _same_device(inds, x, "x")


def switch_glu(g: Geom, slab: torch.Tensor, table, n_experts: int, x: torch.Tensor,
               inds: torch.Tensor) -> torch.Tensor:
    """y [N, K, D] bf16: row (n, k) through the expert in slot table[inds[n, k]]."""
    _need(inds, torch.int32, "inds", 2)
    n, k = inds.shape
    if not _fits(x, torch.bfloat16, (n, g.hidden), inds.get_device()):
        _rows_of(x, n, g, inds)
    y = x.new_empty((n, k, g.hidden))
    if n == 0:
        return y
    ws = moe_workspace(g, n, k, 0, n_experts, x.device)
    check(lib().pmoe_switch_glu(ctypes.byref(g), _ptr(slab), _table_ptr(table, n_experts),
                                n_experts, x.data_ptr(), inds.data_ptr(), n, k, y.data_ptr(),
                                ws.data_ptr(), ws.numel(), _stream()), "pmoe_switch_glu")
    return y


def count_missing(table, ids: torch.Tensor, n_experts: int, counter: torch.Tensor) -> None:
    """counter (device int32 [1]) += routed ids of ``ids`` that ``table``
    (device int32 [E], a tensor or a device address) maps to no slot."""
    _need(ids, torch.int32, "ids")
    _need(counter, torch.int32, "counter", 1)
    check(lib().pmoe_count_missing(_table_ptr(table), _ptr(ids), ids.numel(), n_experts,
                                   _ptr(counter), _stream()), "pmoe_count_missing")


def moe_experts(g: Geom, slab, table, n_experts: int, x, inds, weights, shared_slot: int = -1,
                shared_gate=None) -> torch.Tensor:
    """out [N, D] bf16 = sum_k w[n,k] FFN_{inds[n,k]}(x[n]) (+ shared)."""
    _need(inds, torch.int32, "inds", 2)
    n, k = inds.shape
    dev = inds.get_device()
    if not _fits(x, torch.bfloat16, (n, g.hidden), dev):
        _rows_of(x, n, g, inds)
    if not _fits(weights, torch.float32, (n, k), dev):
        _like(weights, inds, (n, k), "weights", torch.float32)
    if shared_gate is not None and shared_gate.numel() != g.hidden:
        raise ValueError(f"shared_gate must hold {g.hidden} values, got {shared_gate.numel()}")
    out = torch.empty_like(x)
    if n == 0:
        return out
    ws = moe_workspace(g, n, k, int(shared_slot >= 0), n_experts, x.device)
    check(lib().pmoe_moe_experts(ctypes.byref(g), _ptr(slab), _table_ptr(table, n_experts),
                                 n_experts, x.data_ptr(), inds.data_ptr(), weights.data_ptr(), n,
                                 k, int(shared_slot), _ptr(shared_gate), out.data_ptr(),
                                 ws.data_ptr(), ws.numel(), _stream()), "pmoe_moe_experts")
    return out


def combine(y: torch.Tensor, weights: torch.Tensor, shared_y=None, shared_logit=None):
    """out [N, D] bf16 = sum_k weights[n,k] y[n,k] (+ s * shared_y[n]) with
    fp32 accumulation in k order; s = 1 or sigmoid(shared_logit[n])."""
    _need(y, torch.bfloat16, "y", 3)
    _need(weights, torch.float32, "weights", 2)
    n, k, d = y.shape
    if tuple(weights.shape) != (n, k):
        raise ValueError(f"weights must be [{n}, {k}], got {tuple(weights.shape)}")
    if shared_y is not None:
        _need(shared_y, torch.bfloat16, "shared_y", 2)
        if tuple(shared_y.shape) != (n, d):
            raise ValueError("shared_y must be [N, D]")
    if shared_logit is not None:
        _need(shared_logit, torch.float32, "shared_logit")
        if shared_logit.numel() != n:
            raise ValueError("shared_logit must hold N values")
    out = torch.empty((n, d), dtype=torch.bfloat16, device=y.device)
    check(lib().pmoe_combine(_ptr(y), _ptr(weights), n, k, d, _ptr(shared_y), _ptr(shared_logit),
                             _ptr(out), _stream()), "pmoe_combine")
    return out


_STREAM_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _stream_dtype(t, name, dtype=None):
    """The ABI's type of an fp32 or bf16 tensor (of ``dtype``, if given)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name}: expected an fp32 or bf16 tensor")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    return _DTYPES[t.dtype]


def _like(t, ref, shape, name, dtype=None):
    """t is contiguous, of ``shape`` (and ``dtype``), on ref's device."""
    _need(t, t.dtype if dtype is None else dtype, name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected {tuple(shape)}, got {tuple(t.shape)}")
    _same_device(ref, t, name)


def _bf16_rows(x):
    """A new bf16 tensor like the contiguous x (the shorter way where x is bf16)."""
    if x.dtype is torch.bfloat16:
        return torch.empty_like(x)
    return x.new_empty(x.shape, dtype=torch.bfloat16)


def block_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
               unit_offset: bool = False) -> torch.Tensor:
    """h [N, D] bf16: the RMS norm of a residual stream x [N, D] (fp32 or
    bf16) with weight [D] (fp32 or bf16; 1 + weight with unit_offset), the
    input of a block (pmoe_block_norm)."""
    try:
        xd, wd = _STREAM_DTYPES[x.dtype], _STREAM_DTYPES[weight.dtype]
    except (AttributeError, KeyError, TypeError):  # says which it is
        xd, wd = _stream_dtype(x, "x"), _stream_dtype(weight, "weight")
    if not (x.dim() == 2 and x.is_cuda and x.is_contiguous()):
        _need(x, x.dtype, "x", 2)
    n, d = x.shape
    if not (weight.shape == (d,) and weight.get_device() == x.get_device()
            and weight.is_contiguous()):
        _like(weight, x, (d,), "weight")
    h = _bf16_rows(x)
    if n:
        check(lib().pmoe_block_norm(x.data_ptr(), xd, weight.data_ptr(), wd, n, d, eps,
                                    1 if unit_offset else 0, h.data_ptr(), _stream_of(x)),
              "pmoe_block_norm")
    return h


def block_join(residual: torch.Tensor, y: torch.Tensor, weights=None, *, shared_y=None,
               shared_logit=None, post_weight=None, gate=None, gate_sigmoid: bool = False,
               residual_scale: float = 1.0, branch_scale: float = 1.0, next_weight=None,
               eps: float = 1e-6, unit_offset: bool = False, out=None):
    """(out, h): what follows a block, in one pass (pmoe_block_join).

    out [N, D] (residual's type, fp32 or bf16) = residual_scale * residual +
    branch_scale * gate * norm(y); h [N, D] bf16 = norm(out), or None without
    ``next_weight``.  ``y``: a block's outputs bf16 [N, D], or its per-slot
    outputs [N, K, D] with routing ``weights`` fp32 [N, K] (and ``shared_y``,
    ``shared_logit``), combined as ``combine`` does.  ``post_weight`` /
    ``next_weight`` [D] (one type, fp32 or bf16) are the RMS norms'; without
    ``post_weight`` y is not normed.  ``gate`` (fp32 or bf16): [D] per channel,
    [N, 1] per token or [N, D], by itself or its sigmoid.  ``out`` may be
    ``residual`` itself; it overlaps no other input."""
    j = _lib.Join()
    try:
        j.stream_dtype = _STREAM_DTYPES[residual.dtype]
    except (AttributeError, KeyError, TypeError):
        j.stream_dtype = _stream_dtype(residual, "residual")
    if not (residual.dim() == 2 and residual.is_cuda and residual.is_contiguous()):
        _need(residual, residual.dtype, "residual", 2)
    n, d = residual.shape
    dev = residual.get_device()
    bf16 = torch.bfloat16
    if weights is None:
        k = 1
        if not _fits(y, bf16, (n, d), dev):
            _like(y, residual, (n, d), "y", bf16)
    else:
        _need(y, bf16, "y", 3)
        k = y.shape[1]
        if not _fits(y, bf16, (n, k, d), dev):
            _like(y, residual, (n, k, d), "y")
        if not _fits(weights, torch.float32, (n, k), dev):
            _like(weights, residual, (n, k), "weights", torch.float32)
    if shared_y is not None and not _fits(shared_y, bf16, (n, d), dev):
        _like(shared_y, residual, (n, d), "shared_y", bf16)
    if shared_logit is not None:
        _need(shared_logit, torch.float32, "shared_logit")
        _same_device(residual, shared_logit, "shared_logit")
        if shared_y is None or shared_logit.numel() != n:
            raise ValueError("shared_logit must hold N values, beside shared_y")
    if post_weight is not None:
        j.weight_dtype = _stream_dtype(post_weight, "post_weight")
        if not (post_weight.shape == (d,) and post_weight.get_device() == dev
                and post_weight.is_contiguous()):
            _like(post_weight, residual, (d,), "post_weight")
    if next_weight is not None:
        j.weight_dtype = _stream_dtype(next_weight, "next_weight",
                                       None if post_weight is None else post_weight.dtype)
        if not (next_weight.shape == (d,) and next_weight.get_device() == dev
                and next_weight.is_contiguous()):
            _like(next_weight, residual, (d,), "next_weight")
    if gate is not None:
        j.gate_dtype = _stream_dtype(gate, "gate")
        shape = gate.shape
        if shape == (d,):
            j.gate_kind = _lib.GATE_CHANNEL
        elif shape == (n, 1):
            j.gate_kind = _lib.GATE_TOKEN
        elif shape == (n, d):
            j.gate_kind = _lib.GATE_ELEMENT
        else:
            raise ValueError(f"gate: expected {(d,)}, {(n, 1)} or {(n, d)}, got {tuple(shape)}")
        if not (gate.get_device() == dev and gate.is_contiguous()):
            _like(gate, residual, shape, "gate")
        if gate_sigmoid:
            j.gate_sigmoid = 1
    if unit_offset:
        j.unit_offset = 1
    j.residual_scale, j.branch_scale, j.eps = residual_scale, branch_scale, eps
    if out is None:
        out = torch.empty_like(residual)
    elif not _fits(out, residual.dtype, (n, d), dev):
        _like(out, residual, (n, d), "out", residual.dtype)
    h = None
    if next_weight is not None:  # (y is bf16 of that shape where it has no slots)
        h = torch.empty_like(y) if weights is None else _bf16_rows(residual)
    if n:
        check(lib().pmoe_block_join(
            ctypes.byref(j), residual.data_ptr(), y.data_ptr(), _ptr(weights), _ptr(shared_y),
            _ptr(shared_logit), _ptr(post_weight), _ptr(gate), _ptr(next_weight), n, k, d,
            out.data_ptr(), _ptr(h), _stream_of(residual)), "pmoe_block_join")
    return out, h


def route_cfg(scoring: str, n_experts: int, top_k: int, norm_topk_prob: bool = True,
              n_group: int = 1, topk_group: int = 1, routed_scale: float = 1.0) -> RouteCfg:
    rc = RouteCfg()
    rc.scoring = _lib.SCORE_SOFTMAX if scoring == "softmax" else _lib.SCORE_SIGMOID
    rc.n_experts = n_experts
    rc.top_k = top_k
    rc.norm_topk_prob = int(bool(norm_topk_prob))
    rc.n_group = n_group
    rc.topk_group = topk_group
    rc.routed_scale = float(routed_scale)
    return rc


def moe_block(g: Geom, rc: RouteCfg, slab, table, gate_w, x, score_bias=None, logit_bias=None,
              shared_slot: int = -1, shared_gate=None, out=None, inds=None, weights=None,
              ws=None):
    """Route -> dispatch -> experts -> combine in one call.  Returns
    (out [N, D] bf16, inds [N, K] int32, weights [N, K] fp32)."""
    _need(x, torch.bfloat16, "x", 2)
    _need(gate_w, torch.bfloat16, "gate_w", 2)
    n = x.shape[0]
    k = rc.top_k
    dev = x.device
    if x.shape[1] != g.hidden or gate_w.shape[1] != g.hidden or gate_w.shape[0] < rc.n_experts:
        raise ValueError(f"x must be [N, {g.hidden}] and gate_w [{rc.n_experts}, {g.hidden}], got "
                         f"{tuple(x.shape)} and {tuple(gate_w.shape)}")
    if out is None:
        out = torch.empty((n, g.hidden), dtype=torch.bfloat16, device=dev)
    if inds is None:
        inds = torch.empty((n, k), dtype=torch.int32, device=dev)
    if weights is None:
        weights = torch.empty((n, k), dtype=torch.float32, device=dev)
    if ws is None:
        ws = moe_workspace(g, n, k, int(shared_slot >= 0), rc.n_experts, dev)
    check(lib().pmoe_moe_block(ctypes.byref(g), ctypes.byref(rc), _ptr(slab),
                               _table_ptr(table, rc.n_experts),
                               _ptr(gate_w), _ptr(score_bias), _ptr(logit_bias), _ptr(x), n,
                               int(shared_slot), _ptr(shared_gate), _ptr(out), _ptr(inds),
                               _ptr(weights), _ptr(ws), ws.numel(), _stream()), "pmoe_moe_block")
    return out, inds, weights
