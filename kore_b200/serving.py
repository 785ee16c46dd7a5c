"""Operators of a serving step around the quantized-linear path, on CUDA tensors of torch's current stream:

* ``qknorm_rope_append`` — per-head norms of queries and keys, half-split rotation and cache append in one pass,
* ``KV4Cache`` — a KV cache held in 4 bits (append, read-back) and ``attend``, the attention that reads it,
* ``sample`` — one token per row of logits with temperature, top-k, top-p and min-p from given uniform numbers.

The reference's decoder loop has an f32 cache, one KV head per query head and a greedy head
(``crates/kore-edge/src/runtime.rs:106-294``).  All arithmetic runs in the CUDA library (``include/kore_b200.h`` states
it down to the roundings); this file checks shapes and moves pointers.  Activations and logits are float32, as
everywhere in this package.
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext

from . import _cabi
from ._cabi import KoreError


def _need(t, name: str, dtype, shape=None, contiguous: bool = True, device=None):
    """t is a CUDA tensor of this type (and shape, -1 = any; and device), or a KoreError in the library's manner"""
    import torch

    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype:
        got = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise KoreError(_cabi.ERR_DTYPE, f"{name}: expected a CUDA {dtype} tensor, got {got}")
    if shape is not None and (t.dim() != len(shape) or any(w not in (-1, g) for w, g in zip(shape, t.shape))):
        raise KoreError(_cabi.ERR_SHAPE, f"{name}: shape mismatch: expected {list(shape)}, got {list(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise KoreError(_cabi.ERR_INVALID, f"{name}: expected a contiguous tensor")
    if device is not None and t.device != device:
        raise KoreError(_cabi.ERR_INVALID, f"{name}: on {t.device}, the other operands are on {device}")
    return t


def _on(device):
    """the library launches on the current device"""
    import torch

    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device) -> int:
    import torch

    return torch.cuda.current_stream(device).cuda_stream


class KV4Cache:
    """K and V of ``n_seqs`` sequences in 4 bits: per (sequence, KV head, position) a row of codes and one (step, lo) pair
    of bfloat16 numbers, 4.25 bits a value for heads of 128 (f32 caches take 32).

    ``k_codes`` / ``v_codes``: int32 [n_seqs, n_kv_heads, max_len, ceil(head_dim / 8)], ``k_steps`` / ``v_steps``: int32
    [n_seqs, n_kv_heads, max_len]; a code c stands for lo + c * step.  ``max_len`` is rounded up to a multiple of 4."""

    def __init__(self, n_seqs: int, n_kv_heads: int, max_len: int, head_dim: int, device: int = 0):
        import torch

        if min(n_seqs, n_kv_heads, max_len) < 1:
            raise KoreError(_cabi.ERR_INVALID, f"KV4Cache: {n_seqs} sequences, {n_kv_heads} KV heads, {max_len} positions")
        max_len = (max_len + 3) // 4 * 4
        dev = torch.device("cuda", device)
        words = int(_cabi.lib().kb_kv4_row_words(head_dim))
        z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
        self._adopt(z(n_seqs, n_kv_heads, max_len, words), z(n_seqs, n_kv_heads, max_len),
                    z(n_seqs, n_kv_heads, max_len, words), z(n_seqs, n_kv_heads, max_len), head_dim)

    @classmethod
    def from_planes(cls, k_codes, k_steps, v_codes, v_steps, head_dim: int) -> "KV4Cache":
        """A cache over planes that the caller keeps (nothing is copied)."""
        self = cls.__new__(cls)
        self._adopt(k_codes, k_steps, v_codes, v_steps, head_dim)
        return self

    def _adopt(self, k_codes, k_steps, v_codes, v_steps, head_dim):
        import torch

        if head_dim < 4 or head_dim > 128 or head_dim % 4:
            raise KoreError(_cabi.ERR_UNSUPPORTED, f"KV4Cache: head_dim {head_dim} must be a multiple of 4 up to 128")
        _need(k_codes, "k_codes", torch.int32, (-1, -1, -1, (head_dim + 7) // 8))
        shape = tuple(k_codes.shape)
        for t, name, want in ((k_steps, "k_steps", shape[:3]), (v_codes, "v_codes", shape), (v_steps, "v_steps", shape[:3])):
            _need(t, name, torch.int32, want, device=k_codes.device)
        if shape[2] % 4 or 0 in shape:
            raise KoreError(_cabi.ERR_UNSUPPORTED, f"KV4Cache: planes of {list(shape)}: the cache length must be a multiple of 4")
        self.k_codes, self.k_steps, self.v_codes, self.v_steps = k_codes, k_steps, v_codes, v_steps
        self.n_seqs, self.n_kv_heads, self.max_len, self.head_dim = shape[0], shape[1], shape[2], int(head_dim)
        self.device = k_codes.device
        self._planes = tuple(t.data_ptr() for t in (k_codes, k_steps, v_codes, v_steps))

    def memory_bytes(self) -> int:
        return sum(t.numel() * 4 for t in (self.k_codes, self.k_steps, self.v_codes, self.v_steps))

    def read(self, cache_rows, k_out=None, v_out=None):
        """The f32 values of cache rows (int64 [n], row = sequence * max_len + position; zeros for a row outside the
        cache): K and V, each [n, n_kv_heads, head_dim]."""
        import torch

        _need(cache_rows, "cache_rows", torch.int64, (-1,), device=self.device)
        n = cache_rows.shape[0]
        shape = (n, self.n_kv_heads, self.head_dim)
        k_out, v_out = (torch.empty(shape, dtype=torch.float32, device=self.device) if o is None
                        else _need(o, "out", torch.float32, shape, device=self.device) for o in (k_out, v_out))
        if n == 0:
            return k_out, v_out
        with _on(self.device):
            _cabi.check(_cabi.lib().kb_kv4_read(*self._planes, cache_rows.data_ptr(), n, self.n_kv_heads, self.head_dim,
                                                self.n_seqs, self.max_len, k_out.data_ptr(), v_out.data_ptr(), _stream(self.device)))
        return k_out, v_out


def qknorm_rope_append(qkv, positions, cache_rows, cos, sin, cache, n_heads: int, *, q_gamma=None, k_gamma=None, eps: float = 1e-5,
                       q_out=None):
    """Norms (where a gamma [head_dim] is given), rotation and append of rows [q | k | v], float32 [n, (n_heads + 2
    n_kv_heads) head_dim] (rows may be strided).  positions int32 [n], cache_rows int64 [n] (sequence * max_len +
    position; a negative one is padding and appends nothing), cos/sin float32 [max_pos, head_dim / 2].

    ``cache`` is a KV4Cache or a pair (k, v) of float32 caches [n_seqs, n_kv_heads, max_len, head_dim].  Returns the
    queries, float32 [n, n_heads, head_dim].  Two tokens of one call must not name the same cache row."""
    import torch

    f32 = torch.float32
    four = isinstance(cache, KV4Cache)
    if four:
        n_seqs, n_kv, lmax, hd, dev = cache.n_seqs, cache.n_kv_heads, cache.max_len, cache.head_dim, cache.device
    else:
        k, v = cache
        _need(k, "k cache", f32, (-1, -1, -1, -1))
        n_seqs, n_kv, lmax, hd = k.shape
        dev = k.device
        _need(v, "v cache", f32, tuple(k.shape), device=dev)
    _need(qkv, "qkv", f32, (-1, (n_heads + 2 * n_kv) * hd), contiguous=False, device=dev)
    n, width = qkv.shape
    if width and qkv.stride(1) != 1 or (n > 1 and qkv.stride(0) < width):
        qkv = qkv.contiguous()
    ld = qkv.stride(0) if n > 1 else width
    _need(positions, "positions", torch.int32, (n,), device=dev)
    _need(cache_rows, "cache_rows", torch.int64, (n,), device=dev)
    _need(cos, "cos", f32, (-1, hd // 2), device=dev)
    _need(sin, "sin", f32, tuple(cos.shape), device=dev)
    for g, name in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
        if g is not None:
            _need(g, name, f32, (hd,), device=dev)
    if q_out is None:
        q_out = torch.empty((n, n_heads, hd), dtype=f32, device=dev)
    else:
        _need(q_out, "q_out", f32, (n, n_heads, hd), device=dev)
    if n == 0:
        return q_out
    planes = cache._planes if four else (k.data_ptr(), v.data_ptr())
    fn = _cabi.lib().kb_qknorm_rope_kv4 if four else _cabi.lib().kb_qknorm_rope_kv
    with _on(dev):
        _cabi.check(fn(qkv.data_ptr(), ld, positions.data_ptr(), cache_rows.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                       None if q_gamma is None else q_gamma.data_ptr(), None if k_gamma is None else k_gamma.data_ptr(),
                       C.c_float(eps), n, n_heads, n_kv, hd, n_seqs, lmax, q_out.data_ptr(), *planes, _stream(dev)))
    return q_out


def attend(q, cache: KV4Cache, lens, *, scale: float = 0.0, out=None):
    """Causal attention of the last t tokens of each sequence over a 4-bit cache: q float32 [n_seqs, t, n_heads, head_dim]
    (or [n_seqs, n_heads, head_dim], t = 1), lens int32 [n_seqs] the cache positions up to and including the last of the t
    tokens.  Token i sees the positions below lens - (t - 1 - i); one that sees none gives zeros.  scale 0 is
    1 / sqrt(head_dim).  Returns float32 of q's shape."""
    import torch

    hd, dev = cache.head_dim, cache.device
    _need(q, "q", torch.float32, (cache.n_seqs, -1, hd) if q.dim() == 3 else (cache.n_seqs, -1, -1, hd), contiguous=False, device=dev)
    q = q.contiguous()
    t, heads = (1, q.shape[1]) if q.dim() == 3 else (q.shape[1], q.shape[2])
    _need(lens, "lens", torch.int32, (cache.n_seqs,), device=dev)
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", torch.float32, tuple(q.shape), device=dev)
    if out.numel() == 0:
        return out
    lib = _cabi.lib()
    with _on(dev):
        need = lib.kb_attn_kv4_workspace_bytes(cache.n_seqs, t, heads, cache.n_kv_heads, hd, cache.max_len)
        # torch's allocator orders its reuse by stream and keeps a captured graph's blocks to that graph
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _cabi.check(lib.kb_attn_kv4(q.data_ptr(), *cache._planes, lens.data_ptr(), cache.n_seqs, t, heads, cache.n_kv_heads, hd,
                                    cache.max_len, C.c_float(scale), out.data_ptr(), None if ws is None else ws.data_ptr(), need,
                                    _stream(dev)))
    return out


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, return_logprobs: bool = False, tokens=None):
    """One token per row of logits (float32 [n, vocab], rows may be strided) from one uniform number per row, u float32
    [n] in [0, 1).  Settings are None (temperature 1, filter off) or one value per row: temperature, top_p and min_p
    float32 [n], top_k int32 [n].  A temperature of 0 is greedy.  Top-k and min-p act on the tempered distribution, top-p
    on what they keep.  Returns int64 [n], with return_logprobs also float32 [n]: the log of the token's share of what was
    kept."""
    import torch

    f32 = torch.float32
    _need(logits, "logits", f32, (-1, -1), contiguous=False)
    dev = logits.device
    n, vocab = logits.shape
    if logits.stride(1) != 1 and vocab > 1 or (n > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    _need(u, "u", f32, (n,), device=dev)
    ptrs = []
    for t, name, dt in ((temperature, "temperature", f32), (top_k, "top_k", torch.int32), (top_p, "top_p", f32), (min_p, "min_p", f32)):
        ptrs.append(None if t is None else _need(t, name, dt, (n,), device=dev).data_ptr())
    if tokens is None:
        tokens = torch.empty(n, dtype=torch.int64, device=dev)
    else:
        _need(tokens, "tokens", torch.int64, (n,), device=dev)
    logprobs = torch.empty(n, dtype=f32, device=dev) if return_logprobs else None
    if n == 0:
        return (tokens, logprobs) if return_logprobs else tokens
    with _on(dev):
        _cabi.check(_cabi.lib().kb_sample(logits.data_ptr(), n, vocab, logits.stride(0) if n > 1 else vocab, *ptrs, u.data_ptr(),
                                          tokens.data_ptr(), None if logprobs is None else logprobs.data_ptr(), _stream(dev)))
    return (tokens, logprobs) if return_logprobs else tokens
