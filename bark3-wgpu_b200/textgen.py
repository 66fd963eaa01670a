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
by KvCache.check().  The calls have no backward: an input that requires a
gradient is refused unless gradients are off (torch.no_grad()).
"""
from __future__ import annotations

import ctypes

from . import B3_EINVAL, B3_ESTATE, B3_ETIMEOUT, PKG_DIR, B3Error, lib

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


def _load():
    """The torch side of the calls (csrc/textgen_ext.cpp), bound to the C ABI."""
    import torch  # noqa: F401  (its libraries are what the extension links to)

    try:
        from . import _textgen
    except ImportError as e:
        raise B3Error(B3_ESTATE, f"the torch side of text generation is not built for this interpreter "
                                 f"(run make -C {PKG_DIR} textgen): {e}") from e

    L = lib()
    names = ("b3_kv_append", "b3_kv_attend_workspace", "b3_kv_attend", "b3_sample", "b3_last_error")
    _textgen.bind(B3Error, *(ctypes.cast(getattr(L, n), _P).value for n in names))
    return torch, _textgen


_torch, _ext = _load()

sample = _ext.sample


class KvCache(_ext.Cache):
    """Keys and values of many sequences in 8 bits, in pages of `page_tokens`
    tokens with a scale for each page and key head.

    k, v               (pages, kv_heads, page_tokens, head_dim) float8_e4m3fn
    k_scale, v_scale   (pages, kv_heads) float32, powers of two

    Which pages a sequence has is the caller's page table: (n_seq, width)
    int32, entry j of row i the page of tokens [j * page_tokens,
    (j + 1) * page_tokens) of sequence i; entries past its last token are
    never read.  Calls on one cache are made by one thread at a time.  append()
    and attend() are those of _textgen.Cache."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, device: int = 0):
        torch = _torch
        dev = torch.device("cuda", device)
        shape = (pages, kv_heads, page_tokens, head_dim)
        if min(shape) <= 0:
            raise B3Error(B3_EINVAL, f"cache shape {shape}")
        raw = [torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.ones(shape[:2], dtype=torch.float32, device=dev) for _ in range(2)]
        self._adopt(*raw, *scales)

    @classmethod
    def over(cls, k, v, k_scale, v_scale) -> "KvCache":
        """A cache over the caller's own tensors."""
        self = cls.__new__(cls)
        self._adopt(k, v, k_scale, v_scale)
        return self

    def _adopt(self, k, v, k_scale, v_scale) -> None:
        self._status = _torch.zeros(1, dtype=_torch.int32, device=k.device)
        self._hold(k, v, k_scale, v_scale, self._status)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.device = k.device

    def check(self) -> None:
        """Waits for the GPU, all its streams, and raises for what the calls
        since the last check met that only the GPU could see."""
        _torch.cuda.synchronize(self.device)
        bits = int(self._status.item())
        if not bits:
            return
        self._status.zero_()
        if bits & KV_TIMEOUT:
            raise B3Error(B3_ETIMEOUT, "a bounded wait inside the attention ran out")
        what = [s for bit, s in ((KV_BAD_LENGTH, "cu_q or kv_lens out of range"),
                                 (KV_BAD_PAGE, "a page number outside the cache"),
                                 (KV_BAD_POSITION, "a position outside the cos / sin table")) if bits & bit]
        raise B3Error(B3_EINVAL, ", ".join(what))

    def values(self, page: int):
        """The (kv_heads, page_tokens, head_dim) float32 keys and values that a page stands for."""
        return (self.k[page].float() * self.k_scale[page][:, None, None],
                self.v[page].float() * self.v_scale[page][:, None, None])

