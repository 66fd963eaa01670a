"""Text generation beside the encoder: a paged 8-bit cache of keys and values,
the attention that reads it, and the choice of the next token.

    cache = KvCache(pages, kv_heads, head_dim)
    q = cache.append(q, k, v, cu_q, kv_lens, page_table, q_norm=..., k_norm=..., cos=..., sin=...)
    out = cache.attend(q, cu_q, kv_lens, page_table, max_q=1)
    ids, logprob = sample(logits, uniform, temperature=..., top_k=..., top_p=..., min_p=...)

Everything is a torch tensor on one GPU.  The calls enqueue their work on
torch's current stream of that GPU and return; they can be captured in a CUDA
graph.  What they compute is written down at b3_kv_cache, b3_kv_append,
b3_kv_attend and b3_sample in include/bark3_b200.h; a bad argument raises
B3Error(B3_EINVAL), lengths or page numbers that only the GPU sees are reported
by KvCache.check().
"""
from __future__ import annotations

import ctypes
import functools
import struct

from . import B3_EINVAL, B3_ETIMEOUT, DTYPE_BF16, DTYPE_F16, DTYPE_F32, B3Error, check, lib

_P, _I32, _I64, _F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float

KV_BAD_LENGTH, KV_BAD_PAGE, KV_BAD_POSITION, KV_TIMEOUT = 1, 2, 4, 8
SAMPLE_MAX_VOCAB = 262144


class _Cache(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("status", _P), ("pages", _I32),
                ("kv_heads", _I32), ("page_tokens", _I32), ("head_dim", _I32)]


class _Batch(ctypes.Structure):
    _fields_ = [("cu_q", _P), ("kv_lens", _P), ("page_table", _P), ("table_stride", _I64), ("table_width", _I32),
                ("n_seq", _I32), ("tokens", _I32)]


class _Append(ctypes.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("q_token_stride", _I64), ("q_head_stride", _I64),
                ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_token_stride", _I64), ("v_head_stride", _I64),
                ("q_norm", _P), ("k_norm", _P), ("cos", _P), ("sin", _P), ("positions", _P), ("eps", _F32),
                ("dtype", _I32), ("out_dtype", _I32), ("q_heads", _I32), ("rot_dim", _I32), ("rot_rows", _I32),
                ("interleaved", _I32)]


class _Attend(ctypes.Structure):
    _fields_ = [("q", _P), ("out", _P), ("lse", _P), ("q_token_stride", _I64), ("q_head_stride", _I64),
                ("scale", _F32), ("dtype", _I32), ("q_heads", _I32), ("max_q", _I32), ("causal", _I32),
                ("window", _I32)]


class _Sample(ctypes.Structure):
    _fields_ = [("logits", _P), ("uniform", _P), ("temperature", _P), ("top_k", _P), ("top_p", _P), ("min_p", _P),
                ("ids", _P), ("logprob", _P), ("row_stride", _I64), ("dtype", _I32), ("rows", _I32), ("vocab", _I32)]


class _Args:
    """Memory of one argument struct, filled by a single pack: `set(...)`
    takes the fields in order, 0 for a NULL pointer, and `at` is its address."""

    _CODES = {_P: "P", _I32: "i", _I64: "q", _F32: "f"}

    def __init__(self, layout):
        self._buf = ctypes.create_string_buffer(ctypes.sizeof(layout))
        pack = struct.Struct("@" + "".join(self._CODES[t] for _, t in layout._fields_))
        self.set = functools.partial(pack.pack_into, self._buf, 0)
        self.at = ctypes.addressof(self._buf)


_torch = None
_DTYPES: dict = {}


def _torch_module():
    global _torch
    if _torch is None:
        import torch

        _torch = torch
        _DTYPES.update({torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16})
    return _torch


def _fail(msg: str):
    raise B3Error(B3_EINVAL, msg)


def _launch(fn, index: int, *args) -> None:
    """fn(*args, stream) on torch's current stream of GPU `index`, with that GPU current."""
    torch = _torch
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        check(rc)


def _vector(t, name, dtype, n, index):
    """Address of a contiguous (n,) tensor on GPU `index`, 0 where there is none."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.dim() != 1 or t.size(0) != n or t.get_device() != index or not t.is_contiguous():
        _fail(f"{name} must be a contiguous {dtype} tensor of {n} on cuda:{index}, "
              f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


class KvCache:
    """Keys and values of many sequences in 8 bits, in pages of `page_tokens`
    tokens with a scale for each page and key head.

    k, v               (pages, kv_heads, page_tokens, head_dim) float8_e4m3fn
    k_scale, v_scale   (pages, kv_heads) float32, powers of two

    Which pages a sequence has is the caller's page table: (n_seq, width)
    int32, entry j of row i the page of tokens [j * page_tokens,
    (j + 1) * page_tokens) of sequence i; entries past its last token are
    never read.  Calls on one cache are made by one thread at a time."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, device: int = 0):
        torch = _torch_module()
        dev = torch.device("cuda", device)
        shape = (pages, kv_heads, page_tokens, head_dim)
        if min(shape) <= 0:
            _fail(f"cache shape {shape}")
        raw = [torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.ones(shape[:2], dtype=torch.float32, device=dev) for _ in range(2)]
        self._hold(*raw, *scales)

    @classmethod
    def over(cls, k, v, k_scale, v_scale) -> "KvCache":
        """A cache over the caller's own tensors."""
        _torch_module()
        self = cls.__new__(cls)
        self._hold(k, v, k_scale, v_scale)
        return self

    def _hold(self, k, v, k_scale, v_scale) -> None:
        torch = _torch
        if k.dim() != 4 or not k.is_cuda:
            _fail("k must be a (pages, kv_heads, page_tokens, head_dim) tensor on a GPU")
        for t, name, dtype, shape in ((k, "k", torch.float8_e4m3fn, k.shape), (v, "v", torch.float8_e4m3fn, k.shape),
                                      (k_scale, "k_scale", torch.float32, k.shape[:2]),
                                      (v_scale, "v_scale", torch.float32, k.shape[:2])):
            if t.dtype is not dtype or t.shape != shape or t.device != k.device or not t.is_contiguous():
                _fail(f"{name} must be a contiguous {dtype} tensor of {tuple(shape)} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.device = k.device
        self._status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._index = k.get_device()
        self._L = lib()
        self._c, self._b, self._app, self._att = (_Args(x) for x in (_Cache, _Batch, _Append, _Attend))
        self._c.set(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self._status.data_ptr(),
                    self.pages, self.kv_heads, self.page_tokens, self.head_dim)
        self._work: dict = {}   # workspace bytes by what they depend on

    def check(self) -> None:
        """Waits for the GPU and raises for what the calls since the last
        check met that only the GPU could see."""
        bits = int(self._status.item())
        if not bits:
            return
        self._status.zero_()
        if bits & KV_TIMEOUT:
            raise B3Error(B3_ETIMEOUT, "a bounded wait inside the attention ran out")
        what = [s for bit, s in ((KV_BAD_LENGTH, "cu_q or kv_lens out of range"),
                                 (KV_BAD_PAGE, "a page number outside the cache"),
                                 (KV_BAD_POSITION, "a position outside the cos / sin table")) if bits & bit]
        _fail(", ".join(what))

    def _batch(self, tokens, cu_q, kv_lens, page_table) -> int:
        i32, index = _torch.int32, self._index
        n = kv_lens.size(0) if kv_lens.dim() == 1 else -1
        cu, lens = _vector(cu_q, "cu_q", i32, n + 1, index), _vector(kv_lens, "kv_lens", i32, n, index)
        if (page_table.dtype is not i32 or page_table.dim() != 2 or page_table.size(0) != n
                or page_table.get_device() != index or page_table.stride(1) != 1):
            _fail(f"page_table must be a ({n}, width) int32 tensor on {self.device} with adjacent entries")
        width = page_table.size(1)
        self._b.set(cu, lens, page_table.data_ptr(), max(page_table.stride(0), width), width, n, tokens)
        return n

    def _rows(self, t, name, tokens, heads, dtype):
        """Address of new rows (tokens, heads, head_dim), heads of any number where `heads` is None."""
        if (t.dtype is not dtype or t.dim() != 3 or t.size(0) != tokens or t.size(2) != self.head_dim
                or (heads is not None and t.size(1) != heads) or t.stride(2) != 1 or t.get_device() != self._index):
            _fail(f"{name} must be ({tokens}, {heads or 'heads'}, {self.head_dim}) {dtype} on {self.device} with "
                  f"adjacent channels, got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")
        return t.data_ptr()

    def _out(self, out, like, dtype):
        if out is None:
            return _torch.empty(like.shape, dtype=dtype, device=self.device)
        if out.shape != like.shape or out.dtype is not dtype or out.get_device() != self._index or not out.is_contiguous():
            _fail(f"out must be a contiguous {dtype} tensor of {tuple(like.shape)} on {self.device}")
        return out

    def append(self, q, k, v, cu_q, kv_lens, page_table, *, q_norm=None, k_norm=None, eps: float = 1e-6, cos=None,
               sin=None, interleaved: bool = False, positions=None, out=None):
        """Norms and rotates the new tokens' q (tokens, q_heads, head_dim) and
        k (tokens, kv_heads, head_dim), stores k and v in the cache and returns
        the queries, ready for attend(): in q's own type, or float16 for
        float32 input.  kv_lens counts the new tokens already.  q, k and v may
        be views of one projection's output."""
        torch, index, f32 = _torch, self._index, _torch.float32
        tokens, dtype = q.size(0), q.dtype
        code = _DTYPES.get(dtype)
        if code is None:
            _fail(f"q must be float32, float16 or bfloat16, got {dtype}")
        at_q = self._rows(q, "q", tokens, None, dtype)
        at_k = self._rows(k, "k", tokens, self.kv_heads, dtype)
        at_v = self._rows(v, "v", tokens, self.kv_heads, dtype)
        self._batch(tokens, cu_q, kv_lens, page_table)
        out_code = DTYPE_F16 if code == DTYPE_F32 else code
        out = self._out(out, q, torch.float16 if code == DTYPE_F32 else dtype)
        if (cos is None) != (sin is None):
            _fail("cos and sin come together")
        at_cos = at_sin = rot_dim = rot_rows = 0
        if cos is not None:
            for t, name in ((cos, "cos"), (sin, "sin")):
                if t.dtype is not f32 or t.dim() != 2 or t.shape != cos.shape or t.get_device() != index or not t.is_contiguous():
                    _fail(f"{name} must be a contiguous float32 (positions, rot_dim / 2) tensor on {self.device}")
            at_cos, at_sin, rot_rows, rot_dim = cos.data_ptr(), sin.data_ptr(), cos.size(0), 2 * cos.size(1)
        self._app.set(at_q, at_k, at_v, out.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                      v.stride(1), _vector(q_norm, "q_norm", f32, self.head_dim, index),
                      _vector(k_norm, "k_norm", f32, self.head_dim, index), at_cos, at_sin,
                      _vector(positions, "positions", torch.int32, tokens, index), eps, code, out_code, q.size(1),
                      rot_dim, rot_rows, interleaved)
        _launch(self._L.b3_kv_append, index, self._c.at, self._b.at, self._app.at)
        return out

    def attend(self, q, cu_q, kv_lens, page_table, *, max_q: int, scale: float | None = None, causal: bool = True,
               window: int = 0, out=None, return_lse: bool = False):
        """Attention of the new tokens' queries (tokens, q_heads, head_dim),
        float16 or bfloat16, over the cached keys and values of their
        sequences.  max_q: an upper bound of any sequence's new tokens.
        scale: 1 / sqrt(head_dim) by default.  Returns out in q's type, with
        return_lse also the (tokens, q_heads) float32 log-sum-exp."""
        torch, index = _torch, self._index
        tokens, heads, dtype = q.size(0), q.size(1), q.dtype
        if dtype is not torch.float16 and dtype is not torch.bfloat16:
            _fail(f"q must be float16 or bfloat16, got {dtype}")
        at_q = self._rows(q, "q", tokens, None, dtype)
        n = self._batch(tokens, cu_q, kv_lens, page_table)
        out = self._out(out, q, dtype)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=self.device) if return_lse else None
        self._att.set(at_q, out.data_ptr(), lse.data_ptr() if return_lse else 0, q.stride(0), q.stride(1),
                      self.head_dim ** -0.5 if scale is None else scale, _DTYPES[dtype], heads, max_q, causal, window)
        key = (n, tokens, heads, max_q)
        need = self._work.get(key)
        if need is None:
            with torch.cuda.device(index):
                need = self._L.b3_kv_attend_workspace(self._c.at, self._b.at, self._att.at)
            if need < 0:
                check(need)
            if len(self._work) >= 1024:
                self._work.clear()
            self._work[key] = need
        # from torch's allocator on the current stream: calls on other streams get other memory
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _launch(self._L.b3_kv_attend, index, self._c.at, self._b.at, self._att.at, work.data_ptr() if need else 0, need)
        return (out, lse) if return_lse else out

    def values(self, page: int):
        """The (kv_heads, page_tokens, head_dim) float32 keys and values that a page stands for."""
        return (self.k[page].float() * self.k_scale[page][:, None, None],
                self.v[page].float() * self.v_scale[page][:, None, None])


def sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """The next token of every row of logits (rows, vocab), float32, float16 or
    bfloat16: (ids int32, logprob float32), each (rows,).  uniform and the
    settings are (rows,) tensors on the logits' GPU (top_k int32, the others
    float32); None leaves a setting off (temperature: 1)."""
    torch = _torch_module()
    if logits.dim() != 2 or not logits.is_cuda or logits.stride(1) != 1 or logits.dtype not in _DTYPES:
        _fail("logits must be a (rows, vocab) float32, float16 or bfloat16 tensor on a GPU with adjacent columns")
    rows, vocab = logits.shape
    dev = logits.device
    if uniform is None:
        _fail("uniform is missing")
    index, f32 = logits.get_device(), torch.float32
    ids = torch.empty(rows, dtype=torch.int32, device=dev)
    logprob = torch.empty(rows, dtype=f32, device=dev)
    a = _Args(_Sample)
    a.set(logits.data_ptr(), _vector(uniform, "uniform", f32, rows, index),
          _vector(temperature, "temperature", f32, rows, index), _vector(top_k, "top_k", torch.int32, rows, index),
          _vector(top_p, "top_p", f32, rows, index), _vector(min_p, "min_p", f32, rows, index), ids.data_ptr(),
          logprob.data_ptr(), max(logits.stride(0), vocab), _DTYPES[logits.dtype], rows, vocab)
    _launch(lib().b3_sample, index, a.at)
    return ids, logprob
