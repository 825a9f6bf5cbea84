"""Paged KV cache for many requests: block tables and slots of a step, the new
tokens' norms, rotation and cache writes, and their attention over the pages
(the C ABI of include/khq_paged.h).

The uncompressed counterpart of the batched decode and of the chunked prefill:
`plan`, `qk_norm_rope` and `attn` are the launchers, one call each, on tensors
that the caller owns; `PageTable` and `PagedLayer` hold those tensors for a
program that serves requests from slots of a batch.  As in `ops`, arguments are
checked on the host before the launch, which goes to the current HIP stream (or
`stream`) of the tensors' device; there is no fallback.
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct

import torch

from . import _lib
from ._lib import KhqError, ptr, stream_handle
from .build import PAGED_CALLS_PATH, PAGED_LIB_PATH

P, I = ctypes.c_void_p, ctypes.c_int

SIGNATURES = {
    "khq_paged_plan": [P, P, P, I, P, P, I, I, I, I, P, P, P, P, P, P, P, P],
    "khq_qk_norm_rope": [P, P, P],
    "khq_paged_attn": [P, P, P],
    "khq_paged_attn_ws_bytes": [I] * 6,
}
# struct khq_pages, khq_rows and khq_attn_rows of include/khq_paged.h
PAGES_STRUCT = struct.Struct("=2Q3q5i4x")
ROWS_STRUCT = struct.Struct("=10Q12qdf8i4x")
ATTN_STRUCT = struct.Struct("=7QQ6qf5i")

MAX_SEQ = 4096  # KHQ_PAGED_MAX_SEQ
_INT32 = torch.int32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_HEAD_DIMS = (64, 128, 256)

_paged = None
# the raw handle of a device's current stream, where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def lib() -> ctypes.CDLL:
    global _paged
    if _paged is None:
        _lib.lib()  # the library that this one is linked to
        if not os.path.exists(PAGED_LIB_PATH):
            raise RuntimeError(
                f"{PAGED_LIB_PATH} is not built; run __graft_entry__.build() (hipcc, gfx950)")
        loaded = ctypes.CDLL(PAGED_LIB_PATH, mode=os.RTLD_NOW | os.RTLD_GLOBAL)
        for name, argtypes in SIGNATURES.items():
            getattr(loaded, name).argtypes = argtypes
        loaded.khq_paged_attn_ws_bytes.restype = ctypes.c_longlong
        _paged = loaded
    return _paged


def _call(name: str, *args, check: bool = True) -> int:
    rc = getattr(_paged or lib(), name)(*args)
    if check and rc != 0:
        raise KhqError(name, rc)
    return rc


# A step's calls are as long as their checks on the host: each check reads an
# argument once and in one condition, and only its failure asks what was wrong.
def _i32(t, n: int, name: str, device: int) -> int:
    """Pointer of a contiguous int32 tensor of n elements on this device."""
    try:
        if (t.dtype is _INT32 and t.numel() == n and t.get_device() == device
                and t.is_contiguous()):
            return t.data_ptr()
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: dtype {t.dtype}, expected torch.int32")
    if t.get_device() != device:
        raise ValueError(f"{name}: on {t.device}, expected cuda:{device}")
    if t.numel() != n:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {n} elements")
    raise ValueError(f"{name}: must be contiguous")


def _table(t, n_seq, device: int):
    """(pointer, rows, width) of a block table i32 [n_seq][pages]."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("table: expected a torch.Tensor")
    shape = t.shape
    if len(shape) != 2 or (n_seq is not None and shape[0] != n_seq) or not 0 < shape[0] <= MAX_SEQ:
        raise ValueError(f"table: shape {tuple(shape)}, expected "
                         f"[{n_seq or f'1 to {MAX_SEQ}'}][pages of a sequence]")
    n, width = shape
    return _i32(t, n * width, "table", device), n, width


def _heads(t, shape, dtype, name: str, device: int):
    """(pointer, token stride, head stride) of a [tokens][heads][dims] tensor whose
    dims are dense; tokens and heads may be strided."""
    try:
        if t.shape == shape and t.dtype is dtype and t.get_device() == device:
            token, head, dim = t.stride()
            if dim == 1:
                return t.data_ptr(), token, head
            raise ValueError(f"{name}: its last dim must be dense")
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name}: on {t.device}, expected cuda:{device}")
    raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _written(at, shape, name: str):
    """Refuses an output (pointer and strides `at`) whose rows share memory, as an expanded
    tensor's do."""
    _, token, head = at
    n, h, d = shape
    # dims inside heads inside tokens, or inside tokens inside heads
    if head >= d and token >= (h - 1) * head + d or token >= d and head >= (n - 1) * token + d:
        return
    by_token = (h == 1 or head >= d) and (n == 1 or token >= (h - 1) * head + d)
    by_head = (n == 1 or token >= d) and (h == 1 or head >= (n - 1) * token + d)
    if n * h * d and not (by_token or by_head):
        raise ValueError(f"{name}: its rows overlap")


def _device(t, name: str) -> int:
    """Index of the current device, the tensor's."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name}: must be a device tensor")
    if device != _current_device():
        raise ValueError(f"{name}: on {t.device}, but the current device is "
                         f"cuda:{_current_device()}")
    return device


def _stream(stream, device: int):
    """Handle of the stream, or of the device's current one (null: None)."""
    if stream is not None or _raw_stream is None:
        return stream_handle(stream)
    return _raw_stream(device) or None


def _pages(k, v, device: int):
    """struct khq_pages of k, v [n_pages][page_size][H_kv][head_dim] (any strides, dims dense)
    and their shape."""
    for t, name in ((k, "k_pages"), (v, "v_pages")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch.Tensor")
        if t.get_device() != device:
            raise ValueError(f"{name}: on {t.device}, expected cuda:{device}")
    dtype = k.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"k_pages: dtype {dtype}, expected float16 or bfloat16")
    shape = k.shape
    if len(shape) != 4 or shape[3] not in _HEAD_DIMS or 0 in shape:
        raise ValueError(f"k_pages: shape {tuple(shape)}, expected "
                         "[pages][page_size][heads][64, 128 or 256]")
    strides = k.stride()
    if v.shape != shape or v.stride() != strides or v.dtype is not dtype:
        raise ValueError("v_pages: shape, strides and dtype must be those of k_pages")
    page, token, head, dim = strides
    kp, vp = k.data_ptr(), v.data_ptr()
    if dim != 1 or (page | token | head) % 8 or (kp | vp) % 16:
        raise ValueError("k_pages, v_pages: dims must be dense, strides and pointers multiples of "
                         "16 bytes")
    n_pages, page_size, h_kv, d = shape
    if n_pages * page_size >= 1 << 31:
        raise ValueError("k_pages: 2^31 slots or more")
    return PAGES_STRUCT.pack(kp, vp, page, token, head, n_pages, page_size, h_kv, d, code), shape


def plan(q_len, kv_len, table, free_pages, state, *, page_size: int, cu_q, seq_kv, kv_out,
         state_out, status, positions, slots, check: bool = True, stream=None) -> int:
    """khq_paged_plan: from the requests' new tokens (q_len i32 [n_seq]; < 0: ended) and the
    tokens they hold, their new pages, and each batch row's position and slot.  table
    [n_seq][pages], free_pages [n_pages] and state [2] (first free entry, free pages) are the
    cache's bookkeeping; kv_out and state_out may be kv_len and state."""
    device = _device(q_len, "q_len")
    n_seq = q_len.numel()
    table_p, _, width = _table(table, n_seq, device)
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    for t, name in ((free_pages, "free_pages"), (positions, "positions")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch.Tensor")
    n_pages, n_tok = free_pages.numel(), positions.numel()
    return _call("khq_paged_plan", _i32(q_len, n_seq, "q_len", device),
                 _i32(kv_len, n_seq, "kv_len", device), table_p, width,
                 _i32(free_pages, n_pages, "free_pages", device), _i32(state, 2, "state", device),
                 n_seq, n_pages, page_size, n_tok, _i32(cu_q, n_seq + 1, "cu_q", device),
                 _i32(seq_kv, n_seq, "seq_kv", device), _i32(kv_out, n_seq, "kv_out", device),
                 _i32(state_out, 2, "state_out", device), _i32(status, 1, "status", device),
                 _i32(positions, n_tok, "positions", device), _i32(slots, n_tok, "slots", device),
                 _stream(stream, device), check=check)


def qk_norm_rope(q, k, q_out, *, positions=None, pos0: int = 0, q_weight=None, k_weight=None,
                 eps: float = 1e-6, theta: float = 1e7, rotary_dim: int = 64, k_out=None,
                 k_normed=None, v=None, k_pages=None, v_pages=None, slots=None,
                 round_norm: bool = False, check: bool = True, stream=None) -> int:
    """khq_qk_norm_rope: RMS norm of each head of q [n][H_q][D] and k [n][H_kv][D], then the
    half-split rotation of their first rotary_dim dims to `positions` (i32 [n]; None: pos0 and
    on).  Queries go to q_out (q itself will do), keys to k_out and, with pages, to row i's
    slot slots[i], as its values v do; k_normed takes the keys before the rotation.  q or k may
    be None."""
    first = q if q is not None else k
    device = _device(first, "q" if q is not None else "k")
    dt = first.dtype
    if dt not in _DTYPES:
        raise TypeError(f"q, k: dtype {dt}, expected float16 or bfloat16")
    if first.dim() != 3 or first.shape[2] not in _HEAD_DIMS:
        raise ValueError(f"q, k: shape {tuple(first.shape)}, expected "
                         "[tokens][heads][64, 128 or 256]")
    n, _, d = first.shape
    none = (0, 0, 0)
    q_at = q_out_at = k_at = k_out_at = k_normed_at = v_at = none
    h_q = h_kv = 0
    if q is not None:
        h_q = q.shape[1]
        q_at = _heads(q, q.shape, dt, "q", device)
        q_out_at = _heads(q_out, q.shape, dt, "q_out", device)
        _written(q_out_at, q.shape, "q_out")
    if k is not None:
        h_kv = k.shape[1] if k.dim() == 3 else 0
        k_at = _heads(k, (n, h_kv, d), dt, "k", device)
        if k_out is not None:
            k_out_at = _heads(k_out, k.shape, dt, "k_out", device)
            _written(k_out_at, k.shape, "k_out")
        if k_normed is not None:
            k_normed_at = _heads(k_normed, k.shape, dt, "k_normed", device)
            _written(k_normed_at, k.shape, "k_normed")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.dtype != torch.float32 or w.shape != (d,)
                              or w.get_device() != device or not w.is_contiguous()):
            raise ValueError(f"{name}: must be float32 [{d}] on cuda:{device}, contiguous")
    pages, slots_p = None, 0
    if (k_pages is None) != (v_pages is None) or (k_pages is None) != (slots is None) or (
            k_pages is None) != (v is None):
        raise ValueError("v, k_pages, v_pages and slots come together")
    if k_pages is not None:
        if k is None:
            raise ValueError("pages without keys")
        pages, shape = _pages(k_pages, v_pages, device)
        if shape[2:] != (h_kv, d) or k_pages.dtype != dt:
            raise ValueError("k_pages: heads, width and dtype must be those of k")
        v_at = _heads(v, k.shape, dt, "v", device)
        slots_p = _i32(slots, n, "slots", device)
    elif k is not None and k_out is None and k_normed is None:
        raise ValueError("keys without k_out, k_normed or pages")
    pos_p = _i32(positions, n, "positions", device) if positions is not None else 0
    if n == 0:  # (empty tensors have no address)
        return 0
    rows = ROWS_STRUCT.pack(
        q_at[0], q_out_at[0], k_at[0], k_out_at[0], k_normed_at[0], v_at[0], ptr(q_weight) or 0,
        ptr(k_weight) or 0, pos_p, slots_p, *q_at[1:], *q_out_at[1:], *k_at[1:], *k_out_at[1:],
        *k_normed_at[1:], *v_at[1:], theta, eps, n, h_q, h_kv, d, rotary_dim, pos0,
        1 if round_norm else 0, _DTYPES[dt])
    return _call("khq_qk_norm_rope", rows, pages, _stream(stream, device), check=check)


def attn(q, k_pages, v_pages, out, *, cu_q, seq_kv, table, max_q: int, scale: float, gate=None,
         workspace=None, check: bool = True, stream=None) -> int:
    """khq_paged_attn: row i of sequence s (rows cu_q[s] .. cu_q[s + 1] - 1 of q [n][H_q][D])
    sees the sequence's first seq_kv[s] - rows + i + 1 tokens, those of pages table[s]; out
    [n][H_q][D], times sigmoid(gate) with a gate.  max_q: the most rows a sequence has (what
    it says too low or high costs only time).  workspace: a device tensor of attn_ws_bytes
    bytes for calls that may run at once with others; None: the library's."""
    device = _device(q, "q")
    pages, (_, _, h_kv, d) = _pages(k_pages, v_pages, device)
    dt, shape = k_pages.dtype, q.shape
    if len(shape) != 3 or shape[2] != d or shape[1] % h_kv or shape[1] == 0:
        raise ValueError(f"q: shape {tuple(shape)}, expected [tokens][a multiple of {h_kv}][{d}]")
    q_p, q_token, q_head = _heads(q, shape, dt, "q", device)
    out_at = out_p, out_token, out_head = _heads(out, shape, dt, "out", device)
    _written(out_at, shape, "out")
    gate_p, gate_token, gate_head = (_heads(gate, shape, dt, "gate", device)
                                     if gate is not None else (0, 0, 0))
    table_p, n_seq, width = _table(table, None, device)
    ws, ws_bytes = 0, 0
    if workspace is not None:
        if workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError(f"workspace: must be contiguous and on cuda:{device}")
        ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    cu_p, kv_p = _i32(cu_q, n_seq + 1, "cu_q", device), _i32(seq_kv, n_seq, "seq_kv", device)
    n_tok, h_q, _ = shape
    if n_tok == 0:
        return 0
    rows = ATTN_STRUCT.pack(q_p, gate_p, out_p, cu_p, kv_p, table_p, ws, ws_bytes, q_token, q_head,
                            gate_token, gate_head, out_token, out_head, scale, n_tok, n_seq, h_q,
                            width, max_q)
    return _call("khq_paged_attn", rows, pages, _stream(stream, device), check=check)


def attn_ws_bytes(n_tok: int, n_seq: int, H_q: int, H_kv: int, head_dim: int, max_q: int) -> int:
    """Workspace bytes of an attn call of these sizes, whatever its lengths."""
    n = (_paged or lib()).khq_paged_attn_ws_bytes(n_tok, n_seq, H_q, H_kv, head_dim, max_q)
    if n < 0:
        raise KhqError("khq_paged_attn_ws_bytes", n)
    return n


def _native(*functions):
    """The functions behind the checks of khq._paged, which take what is as it should be to
    the same C entry in a microsecond and leave the rest to them (here 4 to 8 us)."""
    if _raw_stream is None or not os.path.exists(PAGED_CALLS_PATH):
        return functions
    lib()
    from . import _paged as calls

    calls.init(KhqError, _raw_stream)
    return [functools.update_wrapper(calls.Call(f), f) for f in functions]


plan, qk_norm_rope, attn = _native(plan, qk_norm_rope, attn)


class PageTable:
    """The pages of up to n_seq requests, kept on the device: which pages each holds, the
    free ones, and what a step's layers read (cu_q, seq_kv, positions, slots).  One table
    serves every layer; a step is one launch, with no word to the host."""

    def __init__(self, n_seq: int, max_pages: int, n_pages: int, page_size: int, n_tok: int,
                 device="cuda"):
        if not 0 < n_seq <= MAX_SEQ or min(max_pages, n_pages, page_size, n_tok) <= 0 or max(
                n_pages, max_pages) * page_size >= 1 << 31:
            raise ValueError("PageTable: sizes out of range")
        self.page_size = page_size
        z = dict(device=device, dtype=torch.int32)
        self.table = torch.zeros((n_seq, max_pages), **z)
        self.kv_len = torch.zeros(n_seq, **z)
        self.free_pages = torch.arange(n_pages, **z)
        self.state = torch.tensor([0, n_pages], **z)
        self.cu_q = torch.zeros(n_seq + 1, **z)
        self.seq_kv = torch.zeros(n_seq, **z)
        self.status = torch.zeros(1, **z)
        self.positions = torch.zeros(n_tok, **z)
        self.slots = torch.zeros(n_tok, **z)

    def step(self, q_len, stream=None) -> None:
        """Appends q_len[s] tokens to request s (i32 [n_seq] on the device; 0: idle, < 0:
        ended).  Afterwards status[0] is the number of refused requests."""
        plan(q_len, self.kv_len, self.table, self.free_pages, self.state,
             page_size=self.page_size, cu_q=self.cu_q, seq_kv=self.seq_kv, kv_out=self.kv_len,
             state_out=self.state, status=self.status, positions=self.positions,
             slots=self.slots, stream=stream)


class PagedLayer:
    """One attention layer over a PageTable: its pages, and its step from the projections
    (head norms, partial rotation, cache writes, attention, gate), the many-request
    counterpart of NativeKhqLayer.attention_step without compression."""

    def __init__(self, pages: PageTable, *, H_q: int = 24, H_kv: int = 4, head_dim: int = 256,
                 dtype=torch.float16, rotary_dim: int = 64, theta: float = 1e7,
                 eps: float = 1e-6, q_weight=None, k_weight=None):
        if H_kv <= 0 or H_q <= 0 or H_q % H_kv:
            raise ValueError("H_q must be a multiple of H_kv")
        if head_dim not in _HEAD_DIMS or dtype not in _DTYPES:
            raise ValueError("head_dim must be 64, 128 or 256, dtype float16 or bfloat16")
        self.pages, self.H_q, self.H_kv, self.D = pages, H_q, H_kv, head_dim
        self.rotary_dim, self.theta, self.eps = rotary_dim, theta, eps
        self.q_weight, self.k_weight = q_weight, k_weight
        shape = (pages.free_pages.shape[0], pages.page_size, H_kv, head_dim)
        z = dict(device=pages.table.device, dtype=dtype)
        self.k_pages = torch.zeros(shape, **z)
        self.v_pages = torch.zeros(shape, **z)

    def attention(self, q_gate, k, v, out, scale: float, *, max_q: int, workspace=None,
                  stream=None) -> None:
        """The step's new tokens (after pages.step): q_gate [n][H_q][2 D] (queries, then their
        gates; the queries become the rotated ones), k, v [n][H_kv][D] -> out [n][H_q][D]."""
        t = self.pages
        if q_gate.dim() != 3 or q_gate.shape[1:] != (self.H_q, 2 * self.D):
            raise ValueError(f"q_gate: shape {tuple(q_gate.shape)}, expected "
                             f"[n][{self.H_q}][{2 * self.D}]")
        q, gate = q_gate[..., :self.D], q_gate[..., self.D:]
        n = q.shape[0]
        if n > t.slots.shape[0]:
            raise ValueError(f"q_gate: {n} rows, the table's step has {t.slots.shape[0]}")
        qk_norm_rope(q, k, q, positions=t.positions[:n], q_weight=self.q_weight,
                     k_weight=self.k_weight, eps=self.eps, theta=self.theta,
                     rotary_dim=self.rotary_dim, v=v, k_pages=self.k_pages,
                     v_pages=self.v_pages, slots=t.slots[:n], stream=stream)
        attn(q, self.k_pages, self.v_pages, out, cu_q=t.cu_q, seq_kv=t.seq_kv, table=t.table,
             max_q=max_q, scale=scale, gate=gate, workspace=workspace, stream=stream)
