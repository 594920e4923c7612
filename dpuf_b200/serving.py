"""Serving operators over a paged key/value cache, on torch tensors of one GPU: rotary positions
fused with the cache's append, attention of new tokens over the cache, and sampling.

They run in libdpuf_cuda.so (`dpuf_cuda_rope_append`, `dpuf_cuda_paged_attention`,
`dpuf_cuda_sample_rows` in include/dpuf_cuda.h, which also states the formulas); this module
checks arguments, allocates outputs and passes device pointers.  Calls enqueue on torch's current
stream of the tensors' device, do not synchronise, and can be captured in a CUDA graph.  Arguments
that do not fit raise ValueError or TypeError, a failed launch RuntimeError.  There is no fallback.

`paged_attention` needs a workspace (39 MB), and calls that share one must not overlap.  Without one
given, a call uses that of the current stream, whose calls follow each other (kept for as long as the
program runs), and a call that `torch.cuda.graph` captures one that its graph has for itself: graphs
may be replayed on any streams, at once too (except where they share a memory pool).  A program that
captures in another way, or wants `attention_check` to see a graph's calls, passes its own from
`attention_workspace`.

One decoding step of a batch, per layer and at its end:

    q = rope_append(cache, page_table, q, k, v, cos, sin, seq, pos)
    o = paged_attention(cache, page_table, q, q_start, kv_len, max_q=1)
    ...
    ids, probs = sample(logits, u, temperature, top_k, top_p, min_p)
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import engine

_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # DPUF_TYPE_*
_KV = struct.Struct("=2Q3q6i")             # DpufPagedKv
_ROPE = struct.Struct("=Qq3Q6qQ2Q2Q10i")   # DpufRopeAppendArgs after its kv
_ATTN = struct.Struct("=QqQ2qQ2QQq9if")    # DpufPagedAttentionArgs after its kv
_INT = torch.int32
_FLOAT = torch.float32

_typed = None
_workspaces: dict = {}  # (device, stream) -> workspace of paged_attention (tensor, address, bytes)
_captured: dict = {}    # (device, stream) -> (capture, such a workspace) of the graph captured on it last
_ZEROED = 8192          # DPUF_PAGED_ATTENTION_ZEROED


def _lib():
    global _typed
    if _typed is None:
        lib = engine.cuda_lib()
        lib.dpuf_cuda_rope_append.restype = ctypes.c_int32
        lib.dpuf_cuda_rope_append.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        lib.dpuf_cuda_paged_attention.restype = ctypes.c_int32
        lib.dpuf_cuda_paged_attention.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        lib.dpuf_cuda_paged_attention_workspace.restype = ctypes.c_int64
        lib.dpuf_cuda_paged_attention_workspace.argtypes = []
        lib.dpuf_cuda_paged_attention_status.restype = ctypes.c_int32
        lib.dpuf_cuda_paged_attention_status.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
        lib.dpuf_cuda_stream_capture_id.restype = ctypes.c_uint64
        lib.dpuf_cuda_stream_capture_id.argtypes = [ctypes.c_void_p]
        lib.dpuf_cuda_sample_rows.restype = ctypes.c_int32
        lib.dpuf_cuda_sample_rows.argtypes = ([ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32,
                                               ctypes.c_int32] + [ctypes.c_void_p] * 8)
        _typed = lib
    return _typed


# torch.cuda.current_stream() and current_device() build objects; these return the numbers
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_capturing = torch._C._cuda_isCurrentStreamCapturing if hasattr(torch._C, "_cuda_isCurrentStreamCapturing") else (
    torch.cuda.is_current_stream_capturing)
_raw_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _call(fn, device: int, *args) -> None:
    """Calls fn(*args, current stream) with `device` current."""
    if _raw_device() == device:
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc == 0:
        return
    if rc == -1:
        raise ValueError(engine.last_error())
    raise RuntimeError(f"rc={rc}: {engine.last_error()}")


def _check(t: torch.Tensor, name: str, dtype, device: int, dims: int) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}")
    if t.dim() != dims or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with {dims} dimension(s)")


def _check_table(t: torch.Tensor, device: int) -> None:
    if t.dtype is _INT and t.get_device() == device and t.dim() == 2 and t.stride(1) == 1:
        return
    if t.dtype != _INT:
        raise TypeError(f"page_table must be {_INT}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"page_table must be on cuda:{device}")
    raise ValueError("page_table must be [sequences, pages] with neighbouring entries of a row adjacent")


class PagedCache:
    """Pools of pages for keys and values, `[n_pages, n_kv, page_size, head_dim]` each (float32,
    float16 or bfloat16; any strides that are multiples of 16 bytes and the same in both, the last
    dimension contiguous).  Which pages a sequence holds is the caller's page table, int32
    `[sequences, pages]`: entry j holds positions `[j * page_size, (j + 1) * page_size)`, -1 none."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        if k_pages.dtype not in _CODE:
            raise TypeError("a cache is float32, float16 or bfloat16")
        if k_pages.dtype != v_pages.dtype or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
            raise ValueError("k_pages and v_pages must have the same type, shape and strides")
        if k_pages.dim() != 4 or k_pages.stride(3) != 1:
            raise ValueError("pages must be [n_pages, n_kv, page_size, head_dim] with contiguous rows")
        if not k_pages.is_cuda or k_pages.device != v_pages.device:
            raise ValueError("pages must be on one GPU")
        n_pages, n_kv, page_size, head_dim = k_pages.shape
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in [8, 1024]")
        if head_dim < 8 or head_dim > 256 or head_dim % 8:
            raise ValueError("head_dim must be a multiple of 8 up to 256")
        size = k_pages.element_size()
        if any(s * size % 16 for s in k_pages.stride()[:3]) or k_pages.data_ptr() % 16 or v_pages.data_ptr() % 16:
            raise ValueError("the pages' addresses and strides must be multiples of 16 bytes")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.n_kv, self.page_size, self.head_dim = n_kv, page_size, head_dim
        self.dtype, self.device_index = k_pages.dtype, k_pages.get_device()
        self._packed = _KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], _CODE[k_pages.dtype],
                                n_pages, n_kv, page_size, head_dim, 0)

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, page_size: int, head_dim: int, dtype=torch.float16,
              device="cuda") -> "PagedCache":
        shape = (n_pages, n_kv, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def rope_table(n_pos: int, rotary_dim: int, theta: float = 1e6, scaling: str = "none", factor: float = 1.0,
               original_pos: int = 0, low_freq: float = 1.0, high_freq: float = 4.0, beta_fast: float = 32.0,
               beta_slow: float = 1.0, device="cuda"):
    """Cosine and sine tables `[n_pos, rotary_dim / 2]` (float32, computed in 64 bits) for the
    angles pos * f_i, f_i = theta^(-2i / rotary_dim), stretched for long contexts:

    "linear"  f / factor;
    "ntk"     theta * factor^(rotary_dim / (rotary_dim - 2)) in theta's place;
    "yarn"    pairs that turn more than beta_fast times over original_pos positions as they are,
              those that turn less than beta_slow times divided by factor, a ramp between, and
              cosine and sine scaled by 0.1 ln(factor) + 1;
    "llama3"  wavelengths under original_pos / high_freq as they are, over original_pos / low_freq
              divided by factor, a blend between.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if n_pos < 1 or factor <= 0:
        raise ValueError("n_pos and factor must be positive")
    if scaling in ("yarn", "llama3") and original_pos < 1:
        raise ValueError(f"{scaling} needs original_pos")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    gain = 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk needs a rotary_dim over 2")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    freq = theta ** (-i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        turns = original_pos * freq / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling == "llama3":
        turns = original_pos * freq / (2 * math.pi)
        keep = ((turns - low_freq) / (high_freq - low_freq)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling}")
    angle = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (gain * angle.cos()).float(), (gain * angle.sin()).float()


def rope_append(cache: PagedCache, page_table: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                cos: torch.Tensor, sin: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor, interleaved: bool = False,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q `[tokens, n_q, head_dim]` and k `[tokens, n_kv, head_dim]` by the tables' row pos[t]
    and stores the turned k and v at position pos[t] of sequence seq[t]; returns the turned q.

    q, k and v have one type (float32, float16, bfloat16) and may be slices of one tensor (the last
    dimension contiguous); the tables turn the first 2 * cos.shape[1] dimensions of each head.  The
    turned q is `out` (contiguous; of any of the types, e.g. the cache's) or a new tensor of q's
    type.  seq and pos are int32 `[tokens]`; pos < 0 marks padding, whose q is zero and which is
    not stored."""
    dev = cache.device_index
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, head_dim]")
    n, n_q, hd = q.shape
    if hd != cache.head_dim or k.shape != (n, cache.n_kv, hd) or v.shape != (n, cache.n_kv, hd):
        raise ValueError("q, k and v do not fit each other or the cache")
    code = _CODE.get(q.dtype)
    if code is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must be of one type: float32, float16 or bfloat16")
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if qs[2] != 1 or ks[2] != 1 or vs[2] != 1:
        raise ValueError("the last dimension of q, k and v must be contiguous")
    if q.get_device() != dev or k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"q, k and v must be on cuda:{dev}")
    if not (cos.dtype is sin.dtype is _FLOAT and cos.get_device() == sin.get_device() == dev and cos.dim() == 2
            and cos.is_contiguous() and sin.is_contiguous() and cos.shape == sin.shape):
        _check(cos, "cos", _FLOAT, dev, 2)
        _check(sin, "sin", _FLOAT, dev, 2)
        raise ValueError("cos and sin must have one shape")
    if not (seq.dtype is pos.dtype is _INT and seq.get_device() == pos.get_device() == dev and seq.is_contiguous()
            and pos.is_contiguous() and seq.shape == pos.shape == (n,)):
        _check(seq, "seq", _INT, dev, 1)
        _check(pos, "pos", _INT, dev, 1)
        raise ValueError("seq and pos must have one entry a token")
    _check_table(page_table, dev)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError("out must be contiguous, of q's shape and on its device")
    elif out.dtype not in _CODE:
        raise TypeError("out must be float32, float16 or bfloat16")
    n_pos, half = cos.shape
    n_seqs, width = page_table.shape
    args = cache._packed + _ROPE.pack(
        page_table.data_ptr(), page_table.stride(0), q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0],
        ks[1], vs[0], vs[1], out.data_ptr(), cos.data_ptr(), sin.data_ptr(), seq.data_ptr(), pos.data_ptr(), n_seqs,
        width, n, n_q, 2 * half, n_pos, bool(interleaved), code, _CODE[out.dtype], 0)
    _call(_lib().dpuf_cuda_rope_append, dev, args)
    return out


def attention_workspace(device: int | None = None) -> torch.Tensor:
    """A workspace for `paged_attention`'s calls, made on the current stream of the device."""
    dev = torch.cuda.current_device() if device is None else device
    ws = torch.empty(_lib().dpuf_cuda_paged_attention_workspace(), dtype=torch.uint8, device=f"cuda:{dev}")
    ws[:_ZEROED].zero_()
    return ws


def _given(ws: torch.Tensor, device: int) -> tuple:
    _check(ws, "workspace", torch.uint8, device, 1)
    if ws.data_ptr() % 16 or ws.numel() < _lib().dpuf_cuda_paged_attention_workspace():
        raise ValueError("workspace is not one of attention_workspace()")
    return ws, ws.data_ptr(), ws.numel()


def _workspace(device: int) -> tuple:
    """The workspace (tensor, address, bytes) of the current stream, or of the capture that it is in."""
    stream = _raw_stream(device)
    key = (device, stream)
    if _raw_device() != device or _capturing():  # (it asks the current device's stream)
        capture = _lib().dpuf_cuda_stream_capture_id(stream)
        if capture:
            found = _captured.get(key)
            # held until the stream's next call after the capture: the graph's pool has the memory, and
            # nothing else captured into the graph may get it
            if found is None or found[0] != capture:
                ws = attention_workspace(device)
                found = _captured[key] = (capture, (ws, ws.data_ptr(), ws.numel()))
            return found[1]
    if _captured:
        _captured.pop(key, None)
    found = _workspaces.get(key)
    if found is None:
        ws = attention_workspace(device)
        found = _workspaces[key] = (ws, ws.data_ptr(), ws.numel())
    return found


def paged_attention(cache: PagedCache, page_table: torch.Tensor, q: torch.Tensor, q_start: torch.Tensor,
                    kv_len: torch.Tensor, max_q: int, scale: float | None = None, causal: bool = True, window: int = 0,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q `[tokens, n_q, head_dim]` over the cache; returns `[tokens, n_q, head_dim]`.

    Sequence s (row s of page_table) has the new tokens q_start[s] .. q_start[s + 1] (int32
    `[sequences + 1]`, ascending), which are the last of its kv_len[s] (int32) positions and have been
    appended; tokens before q_start[0] and from the last entry on are padding and get zeros.  max_q, the
    most new tokens of a sequence, chooses the kernel (results differ by rounding alone).  A token at position
    p sees the positions up to p (all kv_len[s] where not causal), with `window` > 0 the last `window`
    of them; one that sees nothing gets zeros.
    n_q is a multiple of the cache's heads.  q is float32 or of the cache's type and may be a slice
    (the last dimension contiguous, strides multiples of 16 bytes).  scale defaults to
    head_dim^-0.5.  The result is `out` (contiguous; q's type or float32) or a new tensor of q's
    type.  workspace is one of `attention_workspace` that no call or replay in flight uses; without it
    the call uses its stream's, or its graph's."""
    dev = cache.device_index
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        raise ValueError("q must be [tokens, n_q, head_dim] with the cache's head_dim")
    n, n_q, hd = q.shape
    code = _CODE.get(q.dtype)
    if code is None or (code != 0 and q.dtype != cache.dtype):
        raise TypeError("q must be float32 or of the cache's type")
    qs = q.stride()
    if qs[2] != 1:
        raise ValueError("the last dimension of q must be contiguous")
    if q.get_device() != dev:
        raise ValueError(f"q must be on cuda:{dev}")
    _check_table(page_table, dev)
    n_seqs, width = page_table.shape
    if not (q_start.dtype is kv_len.dtype is _INT and q_start.get_device() == kv_len.get_device() == dev
            and q_start.is_contiguous() and kv_len.is_contiguous() and q_start.shape == (n_seqs + 1,)
            and kv_len.shape == (n_seqs,)):
        _check(q_start, "q_start", _INT, dev, 1)
        _check(kv_len, "kv_len", _INT, dev, 1)
        raise ValueError("q_start must have one entry more than page_table has rows, kv_len as many")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError("out must be contiguous, of q's shape and on its device")
    elif out.dtype != q.dtype and out.dtype != _FLOAT:
        raise TypeError("out must be float32 or of q's type")
    _, ws, ws_bytes = _workspace(dev) if workspace is None else _given(workspace, dev)
    args = cache._packed + _ATTN.pack(
        page_table.data_ptr(), page_table.stride(0), q.data_ptr(), qs[0], qs[1], out.data_ptr(), q_start.data_ptr(),
        kv_len.data_ptr(), ws, ws_bytes, n_seqs, width, n, n_q, max_q, bool(causal), window, code,
        _CODE[out.dtype], hd ** -0.5 if scale is None else scale)
    _call(_lib().dpuf_cuda_paged_attention, dev, args)
    return out


def attention_check(device: int | None = None, workspace: torch.Tensor | None = None) -> None:
    """Waits for the current stream and raises RuntimeError if a bounded wait inside a `paged_attention`
    call on the workspace (without one, the stream's) gave up since the last check: the outputs of that
    call and of those after it are undefined.  The workspace is then ready for use again."""
    dev = torch.cuda.current_device() if device is None else device
    ws = _workspace(dev) if workspace is None else _given(workspace, dev)
    _call(_lib().dpuf_cuda_paged_attention_status, dev, ws[1])


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
           min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token a row of logits `[rows, vocab]` (float32, float16 or bfloat16) from the uniforms
    u `[rows]` in [0, 1): ids (int32) and the share of the kept weight that each id has (float32).

    temperature, top_p, min_p (float32) and top_k (int32) are `[rows]` or None (1, 1, 0 and 0: no
    filter).  Of the entries by logit (equal ones by index) the first top_k are kept, of these the
    shortest prefix that holds top_p of their weight, of these the ones with at least min_p of the
    maximum's weight; u picks along the kept ones in index order.  A temperature <= 0 takes the
    first maximum; a row without an entry above -inf gives -1."""
    code = _CODE.get(logits.dtype)
    if code is None:
        raise TypeError("logits must be float32, float16 or bfloat16")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be [rows, vocab] with contiguous rows")
    if not logits.is_cuda:
        raise ValueError("logits must be on a GPU")
    dev = logits.get_device()
    rows, vocab = logits.shape
    if u is None:
        raise TypeError("u is needed")

    def row_values(t, name, dtype):
        if t is None:
            return None
        if not (t.dtype is dtype and t.get_device() == dev and t.is_contiguous() and t.shape == (rows,)):
            _check(t, name, dtype, dev, 1)
            raise ValueError(f"{name} must have one entry a row")
        return t.data_ptr()

    values = (row_values(u, "u", _FLOAT), row_values(temperature, "temperature", _FLOAT),
              row_values(top_k, "top_k", _INT), row_values(top_p, "top_p", _FLOAT), row_values(min_p, "min_p", _FLOAT))
    probs = torch.empty_like(u)
    ids = torch.empty_like(u, dtype=_INT)
    _call(_lib().dpuf_cuda_sample_rows, dev, logits.data_ptr(), code, logits.stride(0), rows, vocab,
          *values, ids.data_ptr(), probs.data_ptr())
    return ids, probs
