"""A memory bank for many requests in one pool of pages, held in 8 bits (include/rmem_hip.h, "paged 8-bit bank").

The dense banks of ``rmem_amd.lstt`` / ``lstt_aot`` hold one clip each, four bytes per element, every slot of one geometry.  Here
requests of any length share a pool; a step is

    p = plan(ctx, add, table, free, state, page=pool.page, rows=T)     # pages, slots and row offsets, on the device
    append(pool, k, v, p.slots)                                        # the new tokens, 8 bits
    out, lse = attend(pool, q, p.cu, p.lens, table, start=p.start, with_lse=True)   # each request's rows over its pages

and ``gather`` reads tokens back as dense rows.  Nothing is read back to the host and nothing synchronises, so a step can be
captured in a hipGraph.  Calls run on torch's current stream of the pool's device, whichever device is current.  Arguments are
checked on the host (`RmemError`); lengths, slots and page ids live on the device, where values outside the pool are skipped.
The caller orders calls on one pool (one stream, or events between streams), as for any tensor that is updated in place.
There is no backward pass: tensors that require grad are refused where gradients are recorded.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import hip
from .hip import Bank8Args, Bank8AppendArgs, Bank8AttnArgs, Bank8GatherArgs, Bank8PlanArgs, RmemError

CODES = {"int8": 0, "e4m3": 1}
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
PAGES = (32, 64, 128)
DIMS = (32, 64, 128)


def _refuse(what: str):
    raise RmemError("bank8: " + what)


def _need(ok: bool, what: str):
    if not ok:
        _refuse(what)


def _ints(t, name: str, shape: tuple, device) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.shape == shape and t.device == device and t.is_contiguous()):
        _refuse(f"{name} must be a contiguous int32 tensor of shape {shape} on {device}")


def _table(t, reqs: int, page: int, device) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and t.dim() == 2 and t.shape[0] == reqs and
            t.shape[1] > 0 and t.stride(1) == 1 and (reqs == 1 or t.stride(0) >= t.shape[1])):
        _refuse(f"table must be an int32 tensor [{reqs}, pages per request] on {device} with contiguous rows")
    if t.shape[1] * page >= 2 ** 31:
        _refuse("pages per request * page must be below 2^31")


class Pool:
    """The pages: codes `k` [pages, heads, dim/16, page, 16], `v` [pages, heads, page/32, 2, dim, 16] (uint8) and scales
    `k_scale`, `v_scale` [pages, heads] (fp32, positive).  Holds the tensors it is given; `Pool.empty` allocates
    them (zeros, scales 1)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, page: int, code: str = "int8"):
        _need(code in CODES, f"code must be one of {sorted(CODES)}")
        _need(page in PAGES, f"page must be one of {PAGES}")
        for t, n in ((k, "k"), (v, "v")):
            _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous() and t.data_ptr() % 16 == 0,
                  f"{n} must be a contiguous uint8 device tensor, 16-byte aligned")
        _need(k.dim() == 5 and k.shape[3] == page and k.shape[4] == 16, "k must be [pages, heads, dim/16, page, 16]")
        pages, heads, dim = k.shape[0], k.shape[1], k.shape[2] * 16
        _need(dim in DIMS, f"dim must be one of {DIMS}")
        _need(pages > 0 and heads > 0 and pages * page < 2 ** 31, "pages and heads must be positive, pages * page below 2^31")
        _need(tuple(v.shape) == (pages, heads, page // 32, 2, dim, 16) and v.device == k.device,
              "v must be [pages, heads, page/32, 2, dim, 16] on k's device")
        for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _need(isinstance(t, torch.Tensor) and t.dtype == torch.float32 and tuple(t.shape) == (pages, heads) and t.is_contiguous() and
                  t.device == k.device, f"{n} must be a contiguous fp32 tensor [pages, heads] on k's device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.page, self.code, self.pages, self.heads, self.dim, self.device = page, code, pages, heads, dim, k.device
        self.args = Bank8Args(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, page, dim, CODES[code])

    @staticmethod
    def empty(pages: int, heads: int, dim: int, page: int = 64, code: str = "int8", device="cuda") -> "Pool":
        _need(dim in DIMS, f"dim must be one of {DIMS}")
        _need(page in PAGES, f"page must be one of {PAGES}")
        _need(code in CODES, f"code must be one of {sorted(CODES)}")
        zero = 128 if code == "int8" else 0
        z = lambda *s: torch.full(s, zero, dtype=torch.uint8, device=device)
        one = lambda: torch.ones(pages, heads, dtype=torch.float32, device=device)
        return Pool(z(pages, heads, dim // 16, page, 16), z(pages, heads, page // 32, 2, dim, 16), one(), one(), page, code)


class Plan(NamedTuple):
    cu: torch.Tensor        # [reqs + 1] first row of each request
    lens: torch.Tensor      # [reqs] tokens held once the rows are appended
    start: torch.Tensor     # [reqs] position of the first new token, -1: not granted
    slots: torch.Tensor     # [rows] slot of each row, -1: none
    state: torch.Tensor     # [2] ring position and number of the free pages that are left
    status: torch.Tensor    # [2] pages taken, pages missing


# torch's current stream of a device as a raw pointer: what torch.cuda.current_stream(device).cuda_stream returns, without the
# Stream object (3 us of a 15 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, name: str, args) -> None:
    call = getattr(hip.load(), name)
    if torch.cuda.current_device() == device.index:
        hip.check(call(C.byref(args), _raw_stream(device.index)), name)
    else:
        with torch.cuda.device(device):
            hip.check(call(C.byref(args), _raw_stream(device.index)), name)


def plan(ctx: torch.Tensor, add: torch.Tensor, table: torch.Tensor, free: torch.Tensor, state: torch.Tensor, *, page: int, rows: int,
         had: Optional[torch.Tensor] = None, out: Optional[Plan] = None) -> Plan:
    """Block tables, slot map and row offsets of one step (rmem_bank8_plan).

    ctx, add [reqs]: tokens that each request holds and wants added; table [reqs, pages per request]: its pages, extended in
    place; free [ring] with state {position, count}: the free pages (as many places as the pool has pages: one that goes back and
    finds none is lost); rows: rows of the step (at least the sum of add, known to
    the caller who packs them); had [reqs]: tokens held before, where requests ended or were cut -- their pages return to the
    ring in place.  A request whose pages are not to be had is left as it was (start -1, slots -1, counted in status[1]).
    `out` gives the results' tensors (a captured step: out.state may be `state`, out.lens may be `ctx`)."""
    _need(isinstance(ctx, torch.Tensor) and ctx.is_cuda and ctx.dim() == 1 and ctx.numel() > 0, "ctx must be a device tensor [reqs]")
    dev, reqs, rows = ctx.device, ctx.numel(), int(rows)
    _need(page in PAGES, "page must be 32, 64 or 128")
    _need(0 <= rows < 2 ** 31, "rows must not be negative")
    one = (reqs,)
    _ints(ctx, "ctx", one, dev)
    _ints(add, "add", one, dev)
    if had is not None:
        _ints(had, "had", one, dev)
    _table(table, reqs, page, dev)
    _need(isinstance(free, torch.Tensor) and free.dim() == 1 and free.numel() > 0, "free must be a tensor [ring]")
    _ints(free, "free", (free.numel(),), dev)
    _ints(state, "state", (2,), dev)
    sizes = (reqs + 1, reqs, reqs, rows, 2, 2)          # in the order of Plan's fields
    if out is None:
        out = Plan(*torch.empty(sum(sizes), dtype=torch.int32, device=dev).split(sizes))
    else:
        for n, size in zip(Plan._fields, sizes):
            _ints(getattr(out, n), "out." + n, (size,), dev)
    a = Bank8PlanArgs(ctx.data_ptr(), add.data_ptr(), hip.ptr(had), reqs, table.data_ptr(), table.stride(0) if reqs > 1 else table.shape[1],
                      table.shape[1], page, free.data_ptr(), free.numel(), state.data_ptr(), out.state.data_ptr(), out.cu.data_ptr(),
                      out.lens.data_ptr(), out.start.data_ptr(), out.slots.data_ptr(), rows, out.status.data_ptr())
    _call(dev, "rmem_bank8_plan", a)
    return out


def _dense(t, name: str, pool: Pool, heads: int, like: Optional[torch.Tensor] = None) -> None:
    if not (isinstance(t, torch.Tensor) and t.dim() == 3 and t.device == pool.device and t.dtype in TYPES and t.shape[1] == heads and
            t.shape[2] == pool.dim):
        _refuse(f"{name} must be fp32, fp16 or bf16 [rows, {heads}, {pool.dim}] on {pool.device}")
    if t.stride(2) != 1:
        _refuse(f"{name}'s last dimension must be contiguous")
    if like is not None and (t.dtype != like.dtype or t.shape != like.shape):
        _refuse(f"{name} must have its partner's type and shape")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires grad, and codes have none: call under torch.no_grad() or with a detached tensor")


def _apart(t: torch.Tensor) -> bool:
    """Whether no two elements of t [rows, heads, dim] lie in one place: the dimension of the smaller step spans that many steps but
    one and a vector, and the other one steps over at least this."""
    (near, n), (far, m) = sorted(((t.stride(1), t.shape[1]), (t.stride(0), t.shape[0])))
    block = near * (n - 1) + t.shape[2]
    return (n < 2 or near >= t.shape[2]) and (m < 2 or far >= block)


def _workspace(given: Optional[torch.Tensor], need: int, device) -> Optional[torch.Tensor]:
    """Scratch of one call: the caller's, or a new tensor (stream-ordered allocator, or the graph's pool while capturing)."""
    _need(need >= 0, "sizes refused (limits of one call: include/rmem_hip.h)")
    if given is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None
    if not (isinstance(given, torch.Tensor) and given.dtype == torch.uint8 and given.is_contiguous() and given.device == device and
            given.numel() >= need and given.data_ptr() % 16 == 0):
        _refuse(f"workspace must be at least {need} contiguous uint8 on {device}, 16-byte aligned")
    return given


def append(pool: Pool, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, workspace: Optional[torch.Tensor] = None) -> None:
    """Writes new tokens k, v [rows, heads, dim] to the pool's slots [rows] (rmem_bank8_append); rows whose slot is -1 are
    skipped.  A page whose first place is written begins anew, otherwise what lies in front of and between the new tokens is
    kept.  workspace: uint8 scratch of this call alone, allocated where it is not given (8 bytes per page of the pool, only for
    more than 4096 rows)."""
    _need(isinstance(pool, Pool), "pool must be a Pool")
    _dense(k, "k", pool, pool.heads)
    _dense(v, "v", pool, pool.heads, k)
    rows = k.shape[0]
    _need(rows < 1 << 24, "fewer than 2^24 rows per call")
    _ints(slots, "slots", (rows,), pool.device)
    if rows == 0:
        return
    a = Bank8AppendArgs(pool.args, k.data_ptr(), v.data_ptr(), TYPES[k.dtype], k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                        slots.data_ptr(), rows, None, 0)
    ws = _workspace(workspace, hip.load().rmem_bank8_append_workspace(C.byref(a)), pool.device)
    if ws is not None:
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _call(pool.device, "rmem_bank8_append", a)


def gather(pool: Pool, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The tokens at `slots` [rows] as dense k, v [rows, heads, dim] of `dtype` (rmem_bank8_gather); zeros where a slot is -1."""
    _need(isinstance(pool, Pool), "pool must be a Pool")
    _need(dtype in TYPES, "dtype must be fp32, fp16 or bf16")
    _need(isinstance(slots, torch.Tensor) and slots.dim() == 1, "slots must be a tensor [rows]")
    _ints(slots, "slots", (slots.numel(),), pool.device)
    rows = slots.numel()
    _need(rows * pool.heads * pool.dim < 1 << 36, "fewer than 2^36 elements per call")
    ko = torch.empty((rows, pool.heads, pool.dim), dtype=dtype, device=pool.device)
    vo = torch.empty_like(ko)
    if rows:
        _call(pool.device, "rmem_bank8_gather", Bank8GatherArgs(pool.args, slots.data_ptr(), rows, ko.data_ptr(), vo.data_ptr(), TYPES[dtype]))
    return ko, vo


def attend(pool: Pool, q: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, *, max_q: Optional[int] = None,
           causal: bool = True, scale: Optional[float] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
           with_lse: bool = False, workspace: Optional[torch.Tensor] = None, start: Optional[torch.Tensor] = None):
    """Attention of each request's rows over its pages (rmem_bank8_attn).

    q [rows, query heads, dim] (query heads a multiple of the pool's; head h reads kv head h // group); cu [reqs + 1]: request
    r's rows; lens [reqs]: its tokens; table [reqs, pages per request]: their pages.  causal: a request's rows are its last
    tokens and see what is not behind them; otherwise every row sees every token.  A row that sees nothing gets 0 (and -inf).
    start [reqs]: plan's -- the rows of a request that was not granted (start < 0) are not in the bank and see nothing; without it
    they count as the last of the tokens that the request had before.
    scale defaults to 1 / sqrt(dim).  max_q: the largest number of rows of one request where known -- it selects kernels, any
    value is safe.  Rows behind the last request are not written: pass `out` (and `lse` [rows, query heads] fp32) where they
    matter.  workspace: uint8 scratch of this call alone, allocated where it is not given.
    A call that would need 2^24 workgroups (1.4 million single rows of 64 query heads over 8, for instance) is refused: divide it.
    Returns out, or (out, lse) with `with_lse` or `lse`."""
    _need(isinstance(pool, Pool), "pool must be a Pool")
    if not (isinstance(q, torch.Tensor) and q.dim() == 3 and q.shape[1] > 0 and q.shape[1] % pool.heads == 0):
        _refuse(f"q must be [rows, a multiple of {pool.heads} heads, {pool.dim}]")
    _dense(q, "q", pool, q.shape[1])
    _need(isinstance(lens, torch.Tensor) and lens.dim() == 1 and lens.numel() > 0, "lens must be a tensor [reqs]")
    dev, reqs, rows, heads_q = pool.device, lens.numel(), q.shape[0], q.shape[1]
    _ints(lens, "lens", (reqs,), dev)
    _ints(cu, "cu", (reqs + 1,), dev)
    _table(table, reqs, pool.page, dev)
    if start is not None:
        _ints(start, "start", (reqs,), dev)
        lens = lens.masked_fill(start < 0, 0)
    scale = 1.0 / math.sqrt(pool.dim) if scale is None else float(scale)
    _need(0.0 < scale < 3e38, "scale must be positive and finite")
    if out is None:
        out = torch.empty((rows, heads_q, pool.dim), dtype=q.dtype, device=dev)
    else:
        _dense(out, "out", pool, heads_q, q)
        _need(_apart(out), "out's rows and heads must lie apart: the larger step at least the extent of the other dimension")
    if lse is not None:
        _need(isinstance(lse, torch.Tensor) and lse.dtype == torch.float32 and tuple(lse.shape) == (rows, heads_q) and lse.is_contiguous() and
              lse.device == dev, "lse must be a contiguous fp32 tensor [rows, query heads]")
    elif with_lse:
        lse = torch.empty((rows, heads_q), dtype=torch.float32, device=dev)
    a = Bank8AttnArgs(pool.args, q.data_ptr(), out.data_ptr(), hip.ptr(lse), TYPES[q.dtype], q.stride(0), q.stride(1), out.stride(0),
                      out.stride(1), cu.data_ptr(), lens.data_ptr(), reqs, rows, table.data_ptr(),
                      table.stride(0) if reqs > 1 else table.shape[1], table.shape[1], heads_q, rows if max_q is None else min(max(int(max_q), 0), 2 ** 31 - 1),
                      int(bool(causal)), scale, None, 0)
    if rows:
        ws = _workspace(workspace, hip.load().rmem_bank8_attn_workspace(C.byref(a)), dev)
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _call(dev, "rmem_bank8_attn", a)
    return out if lse is None else (out, lse)
