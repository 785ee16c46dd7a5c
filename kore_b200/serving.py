"""Operators of a serving step around the quantized-linear path, on CUDA tensors of torch's current stream:

* ``qknorm_rope_append`` — per-head norms of queries and keys, half-split rotation and cache append in one pass,
* ``KV4Cache`` — a KV cache held in 4 bits (append, read-back) and ``attend``, the attention that reads it,
* ``sample`` — one token per row of logits with temperature, top-k, top-p and min-p from given uniform numbers.

The reference's decoder loop has an f32 cache, one KV head per query head and a greedy head
(``crates/kore-edge/src/runtime.rs:106-294``).  All arithmetic runs in the CUDA library (``include/kore_b200.h`` states
it down to the roundings); this file checks shapes and moves pointers.  Calls whose arguments need nothing else go through a
small native module (``csrc/serving_py.cpp``: checks, results and launch in 5 us); it declines every other one, and what
follows here, which also serves where the module has not been built, copies strided operands, changes the device or says what is wrong.  Activations and logits are float32, as
everywhere in this package.  Results carry no gradient.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os
import warnings

import torch

from . import _build, _cabi
from ._cabi import KoreError

_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64


_native = None


class _Declines:
    """stands for the module where there is none: every call goes the other way"""

    append = read = attend = sample = staticmethod(lambda *args: None)


def native():
    """The module of the calls (raises if it has not been built for this Python and torch)."""
    global _native
    if _native is None or _native is _Declines:
        lib, name, path = _cabi.lib(), "kore_b200_serving", _build.module_path()
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: the module has not been built (run `python -m kore_b200._build`)")
        loader = importlib.machinery.ExtensionFileLoader(name, path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location(name, path, loader=loader))
        loader.exec_module(module)
        module.setup(*(_cabi.address(f) for f in (lib.kb_qknorm_rope_kv, lib.kb_qknorm_rope_kv4, lib.kb_kv4_read, lib.kb_attn_kv4,
                                                   lib.kb_attn_kv4_workspace_bytes, lib.kb_sample)))
        _native = module
    return _native


def _calls():
    """the module, or (with one warning) what declines every call: results are the same, a call takes some 5 to 9 us longer"""
    global _native
    _cabi.lib()  # without the CUDA library there is nothing to call: its error
    try:
        return native()
    except (RuntimeError, ImportError) as e:
        warnings.warn(f"calls of kore_b200.serving go without their native module: {e}", RuntimeWarning, stacklevel=3)
        _native = _Declines
        return _native


def _refuse(t, name, dtype, shape, dev):
    """says which of ``_need``'s conditions t misses"""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype:
        got = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise KoreError(_cabi.ERR_DTYPE, f"{name}: expected a CUDA {dtype} tensor, got {got}")
    if shape is not None and tuple(t.shape) != shape:
        raise KoreError(_cabi.ERR_SHAPE, f"{name}: shape mismatch: expected {list(shape)}, got {list(t.shape)}")
    if dev is not None and t.get_device() != dev:
        raise KoreError(_cabi.ERR_INVALID, f"{name}: on {t.device}, the other operands are on cuda:{dev}")
    raise KoreError(_cabi.ERR_INVALID, f"{name}: expected a contiguous tensor")


def _need(t, name: str, dtype, shape, dev: int):
    """t is a contiguous tensor of this type and shape on this GPU, or a KoreError in the library's manner"""
    try:
        if t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous():
            return t
    except AttributeError:
        pass
    _refuse(t, name, dtype, shape, dev)


def _rows(t, name: str, dtype, want: str, dims: int, dev=None):
    """t is a tensor of this type and number of dimensions on this (or any) GPU, strided as it may be; its device index"""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not dtype:
        _refuse(t, name, dtype, None, dev)
    if t.dim() != dims:
        raise KoreError(_cabi.ERR_SHAPE, f"{name}: shape mismatch: expected {want}, got {list(t.shape)}")
    at = t.get_device()
    if dev is not None and at != dev:
        _refuse(t, name, dtype, None, dev)
    return at


def _run(dev: int, fn, *args):
    """the entry point on the device's current stream; the library launches on the current device"""
    # the handles themselves: torch.cuda.current_stream(dev).cuda_stream and current_device() take 2 us of a 9 us call
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc != _cabi.OK:
        _cabi.check(rc)


def _check_head_dim(head_dim):
    if head_dim < 4 or head_dim > 128 or head_dim % 4:
        raise KoreError(_cabi.ERR_UNSUPPORTED, f"KV4Cache: head_dim {head_dim} must be a multiple of 4 up to 128")


class KV4Cache:
    """K and V of ``n_seqs`` sequences in 4 bits: per (sequence, KV head, position) a row of codes and one (step, lo) pair
    of bfloat16 numbers, 4.25 bits a value for heads of 128 (f32 caches take 32).

    ``k_codes`` / ``v_codes``: int32 [n_seqs, n_kv_heads, max_len, ceil(head_dim / 8)], ``k_steps`` / ``v_steps``: int32
    [n_seqs, n_kv_heads, max_len]; a code c stands for lo + c * step.  ``max_len`` is rounded up to a multiple of 4, at most 2^30."""

    def __init__(self, n_seqs: int, n_kv_heads: int, max_len: int, head_dim: int, device: int = 0):
        if min(n_seqs, n_kv_heads, max_len) < 1:
            raise KoreError(_cabi.ERR_INVALID, f"KV4Cache: {n_seqs} sequences, {n_kv_heads} KV heads, {max_len} positions")
        if max_len > 1 << 30:
            raise KoreError(_cabi.ERR_UNSUPPORTED, f"KV4Cache: {max_len} positions, at most {1 << 30}")
        _check_head_dim(head_dim)
        max_len = (max_len + 3) // 4 * 4
        dev = torch.device("cuda", device)
        words = int(_cabi.lib().kb_kv4_row_words(head_dim))
        z = lambda *shape: torch.zeros(shape, dtype=_I32, device=dev)
        self._adopt(z(n_seqs, n_kv_heads, max_len, words), z(n_seqs, n_kv_heads, max_len),
                    z(n_seqs, n_kv_heads, max_len, words), z(n_seqs, n_kv_heads, max_len), head_dim)

    @classmethod
    def from_planes(cls, k_codes, k_steps, v_codes, v_steps, head_dim: int) -> "KV4Cache":
        """A cache over planes that the caller keeps (nothing is copied)."""
        self = cls.__new__(cls)
        self._adopt(k_codes, k_steps, v_codes, v_steps, head_dim)
        return self

    def _adopt(self, k_codes, k_steps, v_codes, v_steps, head_dim):
        _check_head_dim(head_dim)
        dev = _rows(k_codes, "k_codes", _I32, "[n_seqs, n_kv_heads, max_len, words]", 4)
        shape = tuple(k_codes.shape[:3]) + ((head_dim + 7) // 8,)
        for t, name, want in ((k_codes, "k_codes", shape), (k_steps, "k_steps", shape[:3]), (v_codes, "v_codes", shape),
                              (v_steps, "v_steps", shape[:3])):
            _need(t, name, _I32, want, dev)
        if shape[2] % 4 or 0 in shape:
            raise KoreError(_cabi.ERR_UNSUPPORTED, f"KV4Cache: planes of {list(shape)}: the cache length must be a multiple of 4")
        self._held = (k_codes, k_steps, v_codes, v_steps)
        self.n_seqs, self.n_kv_heads, self.max_len, self.head_dim = shape[0], shape[1], shape[2], int(head_dim)
        self.device = k_codes.device
        self._dev = dev
        self._ws_bytes = {}  # workspace of attend by (query tokens, heads)

    # the planes were checked once and stay: they may be written, not replaced
    k_codes = property(lambda self: self._held[0])
    k_steps = property(lambda self: self._held[1])
    v_codes = property(lambda self: self._held[2])
    v_steps = property(lambda self: self._held[3])

    def _planes(self):
        a, b, c, d = self._held
        return a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr()

    def _workspace(self, t: int, heads: int) -> int:
        """Bytes of workspace of ``attend`` with t query tokens: 0 where no sequence is split, one launch instead of two."""
        need = self._ws_bytes.get((t, heads))
        if need is None:
            with torch.cuda.device(self._dev):
                need = self._ws_bytes[t, heads] = int(_cabi.lib().kb_attn_kv4_workspace_bytes(self.n_seqs, t, heads, self.n_kv_heads, self.head_dim,
                                                                                             self.max_len))
        return need

    def memory_bytes(self) -> int:
        return sum(t.numel() * 4 for t in self._held)

    def read(self, cache_rows, k_out=None, v_out=None):
        """The f32 values of cache rows (int64 [n], row = sequence * max_len + position; zeros for a row outside the
        cache): K and V, each [n, n_kv_heads, head_dim]."""
        done = (_native or _calls()).read(self._held, self.head_dim, cache_rows, k_out, v_out)
        if done is not None:
            return done
        dev = self._dev
        _rows(cache_rows, "cache_rows", _I64, "[n]", 1, dev)
        n = cache_rows.shape[0]
        _need(cache_rows, "cache_rows", _I64, (n,), dev)
        shape = (n, self.n_kv_heads, self.head_dim)
        k_out = self.k_steps.new_empty(shape, dtype=_F32) if k_out is None else _need(k_out, "k_out", _F32, shape, dev)
        v_out = self.k_steps.new_empty(shape, dtype=_F32) if v_out is None else _need(v_out, "v_out", _F32, shape, dev)
        if n:
            _run(dev, _cabi.lib().kb_kv4_read, *self._planes(), cache_rows.data_ptr(), n, self.n_kv_heads, self.head_dim, self.n_seqs,
                 self.max_len, k_out.data_ptr(), v_out.data_ptr())
        return k_out, v_out


def qknorm_rope_append(qkv, positions, cache_rows, cos, sin, cache, n_heads: int, *, q_gamma=None, k_gamma=None, eps: float = 1e-5,
                       q_out=None):
    """Norms (where a gamma [head_dim] is given), rotation and append of rows [q | k | v], float32 [n, (n_heads + 2
    n_kv_heads) head_dim] (rows may be strided).  positions int32 [n], cache_rows int64 [n] (sequence * max_len +
    position; a negative one is padding and appends nothing), cos/sin float32 [max_pos, head_dim / 2].

    ``cache`` is a KV4Cache or a pair (k, v) of float32 caches [n_seqs, n_kv_heads, max_len, head_dim].  Returns the
    queries, float32 [n, n_heads, head_dim].  Two tokens of one call must not name the same cache row."""
    four = isinstance(cache, KV4Cache)
    done = (_native or _calls()).append(qkv, positions, cache_rows, cos, sin, cache._held if four else cache, cache.head_dim if four else 0,
                                        n_heads, q_gamma, k_gamma, eps, q_out)
    if done is not None:
        return done
    if four:
        n_seqs, n_kv, lmax, hd, dev = cache.n_seqs, cache.n_kv_heads, cache.max_len, cache.head_dim, cache._dev
        planes, fn = cache._planes(), _cabi.lib().kb_qknorm_rope_kv4
    else:
        k, v = cache
        dev = _rows(k, "k cache", _F32, "[n_seqs, n_kv_heads, max_len, head_dim]", 4)
        n_seqs, n_kv, lmax, hd = shape = k.shape
        _need(k, "k cache", _F32, shape, dev)
        _need(v, "v cache", _F32, shape, dev)
        planes, fn = (k.data_ptr(), v.data_ptr()), _cabi.lib().kb_qknorm_rope_kv
    _rows(qkv, "qkv", _F32, "[n, width]", 2, dev)
    n, width = qkv.shape
    if width != (n_heads + 2 * n_kv) * hd:
        raise KoreError(_cabi.ERR_SHAPE, f"qkv: shape mismatch: expected [{n}, {(n_heads + 2 * n_kv) * hd}], got {list(qkv.shape)}")
    if not qkv.is_contiguous() and (qkv.stride(1) != 1 or (n > 1 and qkv.stride(0) < width)):
        qkv = qkv.contiguous()
    _need(positions, "positions", _I32, (n,), dev)
    _need(cache_rows, "cache_rows", _I64, (n,), dev)
    max_pos = cos.shape[0] if isinstance(cos, torch.Tensor) and cos.dim() == 2 else 0
    _need(cos, "cos", _F32, (max_pos, hd // 2), dev)
    _need(sin, "sin", _F32, (max_pos, hd // 2), dev)
    gq = None if q_gamma is None else _need(q_gamma, "q_gamma", _F32, (hd,), dev).data_ptr()
    gk = None if k_gamma is None else _need(k_gamma, "k_gamma", _F32, (hd,), dev).data_ptr()
    if q_out is None:
        q_out = qkv.new_empty((n, n_heads, hd))
    else:
        _need(q_out, "q_out", _F32, (n, n_heads, hd), dev)
    if n:
        _run(dev, fn, qkv.data_ptr(), qkv.stride(0) if n > 1 else width, positions.data_ptr(), cache_rows.data_ptr(), cos.data_ptr(),
             sin.data_ptr(), max_pos, gq, gk, eps, n, n_heads, n_kv, hd, n_seqs, lmax, q_out.data_ptr(), *planes)
    return q_out


def attend(q, cache: KV4Cache, lens, *, scale: float = 0.0, out=None):
    """Causal attention of the last t tokens of each sequence over a 4-bit cache: q float32 [n_seqs, t, n_heads, head_dim]
    (or [n_seqs, n_heads, head_dim], t = 1), lens int32 [n_seqs] the cache positions up to and including the last of the t
    tokens.  Token i sees the positions below lens - (t - 1 - i); one that sees none gives zeros.  scale 0 is
    1 / sqrt(head_dim).  Returns float32 of q's shape."""
    done = (_native or _calls()).attend(cache._held, cache.head_dim, q, lens, scale, out)
    if done is not None:
        return done
    hd, dev, n = cache.head_dim, cache._dev, cache.n_seqs
    _rows(q, "q", _F32, f"[{n}, (t,) n_heads, {hd}]", 3 if isinstance(q, torch.Tensor) and q.dim() == 3 else 4, dev)
    shape = q.shape
    if shape[0] != n or shape[-1] != hd:
        raise KoreError(_cabi.ERR_SHAPE, f"q: shape mismatch: expected [{n}, (t,) n_heads, {hd}], got {list(shape)}")
    if not q.is_contiguous():
        q = q.contiguous()
    t, heads = (1, shape[1]) if len(shape) == 3 else (shape[1], shape[2])
    _need(lens, "lens", _I32, (n,), dev)
    out = torch.empty_like(q) if out is None else _need(out, "out", _F32, shape, dev)
    if q.numel() == 0:
        return out
    ws, need = 0, cache._workspace(t, heads)
    if need:  # torch's allocator orders its reuse by stream and keeps a captured graph's blocks to that graph
        block = q.new_empty(need // 4)
        ws = block.data_ptr()
    _run(dev, _cabi.lib().kb_attn_kv4, q.data_ptr(), *cache._planes(), lens.data_ptr(), n, t, heads, cache.n_kv_heads, hd, cache.max_len, scale,
         out.data_ptr(), ws, need)
    return out


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, return_logprobs: bool = False, tokens=None):
    """One token per row of logits (float32 [n, vocab], rows may be strided) from one uniform number per row, u float32
    [n] in [0, 1).  Settings are None (temperature 1, filter off) or one value per row: temperature, top_p and min_p
    float32 [n], top_k int32 [n].  A temperature of 0 is greedy.  Top-k and min-p act on the tempered distribution, top-p
    on what they keep.  Returns int64 [n], with return_logprobs also float32 [n]: the log of the token's share of what was
    kept."""
    done = (_native or _calls()).sample(logits, u, temperature, top_k, top_p, min_p, return_logprobs, tokens)
    if done is not None:
        return done
    dev = _rows(logits, "logits", _F32, "[n, vocab]", 2)
    n, vocab = shape = logits.shape
    if not logits.is_contiguous() and (logits.stride(1) != 1 or (n > 1 and logits.stride(0) < vocab)):
        logits = logits.contiguous()
    row = shape[:1]
    _need(u, "u", _F32, row, dev)
    # the tensors stay referenced by the arguments until the launch: a freed one could be handed out again just below
    pt = None if temperature is None else _need(temperature, "temperature", _F32, row, dev).data_ptr()
    pk = None if top_k is None else _need(top_k, "top_k", _I32, row, dev).data_ptr()
    pp = None if top_p is None else _need(top_p, "top_p", _F32, row, dev).data_ptr()
    pm = None if min_p is None else _need(min_p, "min_p", _F32, row, dev).data_ptr()
    tokens = logits.new_empty(row, dtype=_I64) if tokens is None else _need(tokens, "tokens", _I64, row, dev)
    logprobs = logits.new_empty(row) if return_logprobs else None
    if n:
        _run(dev, _cabi.lib().kb_sample, logits.data_ptr(), n, vocab, logits.stride(0) if n > 1 else vocab, pt, pk, pp, pm,
             u.data_ptr(), tokens.data_ptr(), logprobs.data_ptr() if return_logprobs else None)
    return (tokens, logprobs) if return_logprobs else tokens
