"""Python side of the 8-bit paged KV cache operators (dm_kv8_plan, dm_rope, dm_kv8_append,
dm_kv8_attention of include/dismoen_cuda.h) over torch CUDA tensors.

A host runtime that keeps its own paged cache runs, per step,

    plan = plan_slots(free, state, table, lens, new_lens, max_tokens)      # pages and slots
    q, k = rope(rope_plan, q, k, plan.positions)
    append(cache, k, v, plan.slots)
    out = attention(cache, q, table, plan.seq_lens, plan.cu_new, max_q_len, workspace=ws)

Every call runs on torch's current stream (or `stream`, a cudaStream_t) of the tensors' device
and returns without waiting, so a step may be captured into a CUDA graph (with the outputs
given).  Outputs that are not given are allocated on the stream of the call.  The operators serve:
they have no gradients and refuse tensors that ask for one or carry a forward-mode tangent.
Arguments are checked on the host and raise DmError; what only the device can see goes into an
error word, the call's `err` or one of the device's own, and is raised by `check()`.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

PAGE_TOKENS = 16
MAX_REQUESTS = 8192
FILL_ROWS = 2
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "yarn": 2}
_DTYPES = {torch.bfloat16: _lib.DM_DTYPE_BF16, torch.float32: _lib.DM_DTYPE_F32}
_ERR = 512
_local = threading.local()


def _buffer():
    """This thread's message buffer."""
    buf = getattr(_local, "buf", None)
    if buf is None:
        buf = _local.buf = C.create_string_buffer(_ERR)
    return buf


def _raise(rc: int, buf):
    raise _lib.DmError(rc, buf.value.decode())


def _bad(detail: str):
    raise _lib.DmError(_lib.DM_ERR_INVALID_ARG,
                       '{"error_type":"INVALID_ARG","detail":"%s","stage":"kv8","layer":-1}' % detail)


def _stream(device, stream) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index) if stream is None else stream


def _allocate(device, stream, make, *args):
    """A call's output, on the stream of the call: torch reuses memory in the order of one stream."""
    if stream is None or device.type != "cuda":
        return make(*args)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)):
        return make(*args)


def _ints(device, names, *tensors):
    """int32, contiguous, on the device (None: not given)."""
    for i, t in enumerate(tensors):
        if t is not None and (t.dtype is not torch.int32 or t.device != device or not t.is_contiguous()):
            _bad(f"{names.split()[i]} must be a contiguous int32 tensor on {device}")
    if device.type != "cuda":
        _bad(f"the tensors must be on a CUDA device (got {device})")


def _rows(name: str, t: torch.Tensor, heads, dim: int, device, dtype):
    """Checks [rows][heads][dim] with contiguous heads; (address, row stride, head stride, rows, heads)."""
    shape, stride = t.shape, t.stride()
    if (len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads) or t.dtype is not dtype
            or t.device != device or (stride[2] != 1 and t.numel())):
        _bad(f"{name} must be [rows][{'heads' if heads is None else heads}][{dim}] {dtype} on {device}, head elements "
             f"contiguous (got {tuple(shape)} {t.dtype} on {t.device})")
    if t.requires_grad and torch.is_grad_enabled():
        _bad(f"{name} asks for a gradient; the operator has none (use torch.no_grad or detach)")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _bad(f"{name} carries a forward-mode gradient; the operator has none (use forward_ad.unpack_dual)")
    return t.data_ptr(), stride[0], stride[1], shape[0], shape[1]


def error_word(device="cuda") -> torch.Tensor:
    """The device error word the operators OR their DM_DEVERR_* bits into."""
    return torch.zeros(1, dtype=torch.int32, device=device)


def check(err: torch.Tensor | None = None, stream=None, device=None) -> None:
    """Waits for the stream, clears the error word and raises DmError when a bit was set.  Without
    `err`: the word of the device (by default the current one) that all calls without `err` share."""
    buf = _buffer()
    if err is not None:
        rc = _lib.load().dm_kv8_status(err.data_ptr(), _stream(err.device, stream), buf, _ERR)
    else:
        with torch.cuda.device(device):
            rc = _lib.load().dm_kv8_status(
                None, torch.cuda.current_stream().cuda_stream if stream is None else stream, buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)


class Kv8Cache:
    """pages uint8 [num_pages][K|V][kv heads][16][head_dim] e4m3 codes, scales fp32
    [num_pages][K|V][kv heads] powers of two; value = code * scale."""

    def __init__(self, pages: torch.Tensor, scales: torch.Tensor):
        if (pages.dim() != 5 or pages.shape[1] != 2 or pages.shape[3] != PAGE_TOKENS or pages.dtype != torch.uint8
                or not pages.is_contiguous() or not pages.is_cuda):
            _bad("pages must be a contiguous uint8 CUDA tensor [num_pages][2][kv heads][16][head_dim]")
        if (scales.shape != pages.shape[:3] or scales.dtype != torch.float32 or not scales.is_contiguous()
                or scales.device != pages.device):
            _bad("scales must be a contiguous float32 tensor [num_pages][2][kv heads] beside the pages")
        self.pages, self.scales = pages, scales
        self.device = pages.device
        self.num_pages, _, self.num_kv_heads, _, self.head_dim = pages.shape
        self._c = _lib.DmKv8Cache(pages.data_ptr(), scales.data_ptr(), self.num_pages, self.num_kv_heads,
                                  self.head_dim, 0)
        self._ref = C.addressof(self._c)

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, device="cuda") -> "Kv8Cache":
        return cls(torch.zeros((num_pages, 2, num_kv_heads, PAGE_TOKENS, head_dim), dtype=torch.uint8, device=device),
                   torch.full((num_pages, 2, num_kv_heads), 2.0 ** -100, dtype=torch.float32, device=device))

    def values(self) -> torch.Tensor:
        """The whole cache as fp32 (a copy)."""
        return self.pages.view(torch.float8_e4m3fn).float() * self.scales[..., None, None]


def free_list(num_pages: int, device="cuda"):
    """(free_pages, free_state) with every page free; page 0 is the first to be taken."""
    pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
    return pages, torch.tensor([num_pages, 0], dtype=torch.int32, device=device)


class SlotPlan(NamedTuple):
    """seq_lens [n], cu_new [n + 1]; slots, positions, requests [max_tokens] (-1 behind the last token)."""
    seq_lens: torch.Tensor
    cu_new: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    requests: torch.Tensor


def plan_slots(free_pages, free_state, block_table, ctx_lens, new_lens, max_tokens: int, *, state_out=None,
               out: SlotPlan | None = None, err=None, stream=None) -> SlotPlan:
    """dm_kv8_plan: pages for the new tokens of every request (new_lens -1 returns a request's
    pages), written into block_table and taken from the free list (free_state in place, or to
    state_out).  `out` may hold the results' tensors; its seq_lens may be ctx_lens."""
    dev = ctx_lens.device
    n = ctx_lens.numel()
    if out is None:
        room = _allocate(dev, stream, ctx_lens.new_empty, 2 * n + 1 + 3 * max_tokens)
        out = SlotPlan(*room.split_with_sizes((n, n + 1, max_tokens, max_tokens, max_tokens)))
    else:
        _ints(dev, "seq_lens cu_new slots positions requests", *out)
        if (out.seq_lens.numel() < n or out.cu_new.numel() < n + 1
                or min(out.slots.numel(), out.positions.numel(), out.requests.numel()) < max_tokens):
            _bad("an output of the plan is too small")
    _ints(dev, "ctx_lens new_lens block_table free_pages free_state state_out err", ctx_lens, new_lens, block_table,
          free_pages, free_state, state_out, err)
    if new_lens.numel() != n or block_table.dim() != 2 or block_table.shape[0] < n or free_state.numel() != 2 or \
            (state_out is not None and state_out.numel() != 2):
        _bad("need new_lens [n], block_table [n][width], free_state [2]")
    buf = _buffer()
    rc = _lib.load().dm_kv8_plan(
        n, ctx_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), block_table.shape[1],
        free_pages.data_ptr(), free_pages.numel(), free_state.data_ptr(),
        (free_state if state_out is None else state_out).data_ptr(), out.seq_lens.data_ptr(), out.cu_new.data_ptr(),
        max_tokens, out.slots.data_ptr(), out.positions.data_ptr(), out.requests.data_ptr(),
        None if err is None else err.data_ptr(), _stream(dev, stream), buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)
    return out


class RopePlan:
    """Rotary angles of a head: `rotary_dim` of its `head_dim` elements turn (None: all), in
    "half" or "interleaved" pairs, unscaled or stretched ("linear", "yarn") by `factor` past
    `original_context`."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, *, theta: float = 1e4, layout: str = "half",
                 scaling: str = "none", factor: float = 1.0, original_context: float = 32768, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: float = 0.0):
        if layout not in LAYOUTS or scaling not in SCALINGS:
            _bad(f"unknown layout {layout!r} or scaling {scaling!r}".replace('"', "'"))
        p = _lib.DmRopeParams(head_dim, head_dim if rotary_dim is None else rotary_dim, LAYOUTS[layout],
                              SCALINGS[scaling], theta, factor, original_context, beta_fast, beta_slow,
                              attention_factor)
        self._c = _lib.DmRopePlan()
        self._ref = C.addressof(self._c)
        buf = _buffer()
        rc = _lib.load().dm_rope_plan_init(C.byref(p), C.byref(self._c), buf, _ERR)
        if rc != _lib.DM_OK:
            _raise(rc, buf)
        self.head_dim, self.rotary_dim, self.layout = self._c.head_dim, self._c.rotary_dim, layout
        self.mscale = self._c.mscale

    @property
    def freq(self) -> list[float]:
        return list(self._c.freq[:self.rotary_dim // 2])


def rope(plan: RopePlan, q, k, positions, *, q_out=None, k_out=None, stream=None):
    """dm_rope: rotated q [n][Hq][D] and k [n][Hk][D] (k may be None).  q_out / k_out may be
    q / k themselves; rows at negative positions are skipped."""
    dev, D = positions.device, plan.head_dim
    n = positions.numel()
    _ints(dev, "positions", positions)
    if q.dtype not in _DTYPES:
        _bad(f"q is bf16 or fp32 (got {q.dtype})")
    k = q[:, :0] if k is None else k
    q_out = _allocate(dev, stream, torch.empty_like, q) if q_out is None else q_out
    k_out = _allocate(dev, stream, torch.empty_like, k) if k_out is None else k_out
    q_ptr, q_rs, q_hs, q_rows, hq = _rows("q", q, None, D, dev, q.dtype)
    k_ptr, k_rs, k_hs, k_rows, hk = _rows("k", k, None, D, dev, q.dtype)
    qo_ptr, qo_rs, qo_hs, qo_rows, _ = _rows("q_out", q_out, hq, D, dev, q.dtype)
    ko_ptr, ko_rs, ko_hs, ko_rows, _ = _rows("k_out", k_out, hk, D, dev, q.dtype)
    if not n == q_rows == k_rows == qo_rows == ko_rows:
        _bad(f"{n} positions, but q, k, q_out, k_out have {q_rows}, {k_rows}, {qo_rows}, {ko_rows} rows")
    buf = _buffer()
    rc = _lib.load().dm_rope(
        plan._ref, _DTYPES[q.dtype], n, positions.data_ptr(), q_ptr, q_rs, q_hs, qo_ptr, qo_rs, qo_hs, hq, k_ptr, k_rs,
        k_hs, ko_ptr, ko_rs, ko_hs, hk, _stream(dev, stream), buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)
    return q_out, k_out


def append(cache: Kv8Cache, k, v, slots, *, err=None, stream=None) -> None:
    """dm_kv8_append: k, v [n][kv heads][D] quantised into slots [n] of the cache's pages."""
    n = slots.numel()
    if k.dtype not in _DTYPES:
        _bad(f"k is bf16 or fp32 (got {k.dtype})")
    k_ptr, k_rs, k_hs, k_rows, _ = _rows("k", k, cache.num_kv_heads, cache.head_dim, cache.device, k.dtype)
    v_ptr, v_rs, v_hs, v_rows, _ = _rows("v", v, cache.num_kv_heads, cache.head_dim, cache.device, k.dtype)
    _ints(cache.device, "slots err", slots, err)
    if k_rows < n or v_rows < n:
        _bad(f"{n} slots, k has {k_rows} rows, v {v_rows}")
    buf = _buffer()
    rc = _lib.load().dm_kv8_append(
        cache._ref, _DTYPES[k.dtype], n, k_ptr, k_rs, k_hs, v_ptr, v_rs, v_hs, slots.data_ptr(),
        None if err is None else err.data_ptr(), _stream(cache.device, stream), buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)


def attention_workspace(cache: Kv8Cache) -> torch.Tensor:
    """A zeroed workspace for attention() calls on this cache's geometry; calls that may run
    at the same time need one each."""
    nbytes = C.c_uint64()
    buf = _buffer()
    rc = _lib.load().dm_kv8_attention_workspace(cache._ref, C.byref(nbytes), buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)
    return torch.zeros(nbytes.value, dtype=torch.uint8, device=cache.device)


def attention(cache: Kv8Cache, q, block_table, seq_lens, cu_q=None, max_q_len: int = 1, *, sm_scale=None, out=None,
              lse=None, workspace, err=None, stream=None) -> torch.Tensor:
    """dm_kv8_attention: q [rows][Hq][D] against the cached tokens of each request; rows
    [cu_q[i], cu_q[i + 1]) belong to request i and are its last tokens (cu_q None: one row
    per request).  Rows that no request writes (before cu_q[0], from cu_q[n] on, those of a request
    that is skipped) are left as they were in `out`, and zeros if `out` is not given."""
    dev, D = cache.device, cache.head_dim
    n = seq_lens.numel()
    if q.dtype not in _DTYPES:
        _bad(f"q is bf16 or fp32 (got {q.dtype})")
    q_ptr, q_rs, q_hs, rows, hq = _rows("q", q, None, D, dev, q.dtype)
    flags = 0
    if out is None:
        out, flags = _allocate(dev, stream, torch.empty_like if n else torch.zeros_like, q), FILL_ROWS
    out_ptr, out_rs, out_hs, out_rows, _ = _rows("out", out, hq, D, dev, q.dtype)
    _ints(dev, "block_table seq_lens cu_q err", block_table, seq_lens, cu_q, err)
    if block_table.dim() != 2 or block_table.shape[0] < n or (cu_q is not None and cu_q.numel() < n + 1) or \
            out_rows < rows:
        _bad("need block_table [n][width], cu_q [n + 1] and out of q's shape")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != tuple(q.shape[:2]) or
                            not lse.is_contiguous() or lse.device != dev):
        _bad("lse must be a contiguous float32 [rows][Hq]")
    if workspace.device != dev or not workspace.is_contiguous():
        _bad("the workspace must be a contiguous tensor on the cache's device")
    a = _lib.DmKv8AttnArgs(
        _DTYPES[q.dtype], n, hq, max_q_len, rows, block_table.shape[1], D ** -0.5 if sm_scale is None else sm_scale, flags,
        q_ptr, q_rs, q_hs, out_ptr, out_rs, out_hs, None if lse is None else lse.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), None if err is None else err.data_ptr())
    buf = _buffer()
    rc = _lib.load().dm_kv8_attention(cache._ref, C.addressof(a), _stream(dev, stream), buf, _ERR)
    if rc != _lib.DM_OK:
        _raise(rc, buf)
    return out
