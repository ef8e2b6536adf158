"""Attention on the sm_100a kernels: packed sequences, one new token over a cache, and rows
of a pair representation with a shared bias.

* `packed_attention` -- sequences of different lengths stored one behind the other, grouped
  key / value heads, causal or not; forward and backward.
* `cached_attention` -- its form for single tokens: one query per sequence over a key / value
  cache whose lengths live on the device; no backward.
* `pair_attention`   -- attention of every row of a pair representation, with an additive bias
  that all rows of a batch element share and a mask of the keys (triangle attention, and
  with one row the single representation's attention with pair bias); forward and backward,
  the bias' gradient included.

On CUDA tensors the kernels take fp16 and bf16 with a head dimension that is a multiple of 8
up to 128, and raise `NativeDeclined` for anything else; sums, softmax statistics and
gradients' accumulators are fp32. Elsewhere the formula runs in torch, in fp32. A query that
sees no key gives zeros, and masked keys count as absent whatever K and V hold there. The kernels
have first derivatives in reverse mode only; second ones and tangents (forward mode) are refused.
"""

import ctypes
import math
import threading

import torch

from .. import _lib

_TYPES = (torch.float16, torch.bfloat16)


class AttentionErrorWord:
    """The error words of the attention kernels of one GPU: one on the device, which their waits
    poll, and one in pinned host memory, which a kernel writes only when it gave up on a wait.
    The next call (or `check`) sees that with a plain read; no call copies or synchronises.

    Kernels of other streams give up with the one whose wait expired. So every thread that has
    called before raises once, at its next call or `check`, whichever of them clears the words:
    the GPU's failures are counted, and each thread compares with the count it saw last (in the
    extension, which looks at each call)."""

    def __init__(self, device):
        if torch.cuda.is_current_stream_capturing():
            raise _lib.NativeDeclined("the first attention call on a GPU cannot be captured: warm up before the capture")
        self.dev = torch.zeros(64, dtype=torch.int32, device=device)
        self.host = torch.zeros(16, dtype=torch.int32).pin_memory()
        self.ptr, self.host_ptr = self.dev.data_ptr(), self.host.data_ptr()
        self.word = ctypes.c_int32.from_address(self.host_ptr)
        self.index, self.code, self.lock = self.dev.device.index, 0, threading.Lock()
        torch.cuda.synchronize(device)     # zeroed, whatever stream reads it first
        _lib.torch_ext().set_words(self.index, self.ptr, self.host_ptr)

    def poll(self):
        cleared = False
        if self.word.value:
            if torch.cuda.is_current_stream_capturing():
                self._raise(self.word.value)       # (the words stay set: nothing can be cleared here)
            with self.lock:
                if self.word.value:
                    torch.cuda.synchronize(self.dev.device)   # the kernels that met the error have drained
                    self.code = self.word.value
                    self.dev.zero_()
                    # before the host word: while that is set, other threads' calls come here and wait
                    torch.cuda.synchronize(self.dev.device)
                    _lib.torch_ext().count_failure(self.index)
                    self.word.value = 0
                    cleared = True
        if _lib.torch_ext().missed_failure(self.index) or cleared:
            self._raise(self.code)

    def _raise(self, code):
        raise _lib.NativeKernelError(
            f"a bounded device wait expired in a native attention kernel (code 0x{code:x}: kernel "
            f"{code >> 8}, role {(code >> 4) & 15}, site {code & 15}); attention outputs of this GPU, of any "
            "stream, that were formed since this thread's last call or check are invalid")

    def check(self):
        torch.cuda.synchronize(self.dev.device)
        self.poll()


_ERROR_WORDS = {}
_ERROR_WORDS_LOCK = threading.Lock()


def attention_error_word(device=None):
    """The AttentionErrorWord of a GPU (default: the current one)."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    w = _ERROR_WORDS.get(index)
    if w is None:
        with _ERROR_WORDS_LOCK:      # one per GPU, never replaced: kernels hold its addresses
            w = _ERROR_WORDS.get(index)
            if w is None:
                w = _ERROR_WORDS[index] = AttentionErrorWord(torch.device("cuda", index))
    return w


# --------------------------------------------------------------------------- checks
def _scale(scale, dim):
    s = dim ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(s) and s >= 0):
        raise ValueError(f"scale must be finite and not negative, got {scale}")
    return s


def _same(device, dtype, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, q on {device}")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype}, q {dtype}")


def _heads(q_heads, kv_heads, dim, cuda, dtype):
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"{q_heads} query heads cannot share {kv_heads} key / value heads")
    if dim < 1:
        raise ValueError("the head dimension is empty")
    if not cuda:
        return
    if dtype not in _TYPES:
        raise _lib.NativeDeclined(f"attention kernels take fp16 and bf16, got {dtype}")
    if dim % 8 or dim > 128:
        raise _lib.NativeDeclined(f"attention kernels take head dimensions that are multiples of 8 up to 128, got {dim}")
    if q_heads // kv_heads > 128:
        raise _lib.NativeDeclined("at most 128 query heads per key / value head")


def _in_place(t):
    """`t` if the kernels can read it where it is (dense, 16-byte aligned vectors of the last
    dimension, any other strides of whole vectors), else a contiguous copy."""
    st, sh = t.stride(), t.shape
    if st[-1] != 1 or t.data_ptr() % 16:
        return t.contiguous() if not t.is_contiguous() or t.data_ptr() % 16 == 0 else t.clone()
    for s, n in zip(st[:-1], sh[:-1]):
        if n > 1 and (s <= 0 or s % 8):
            return t.contiguous()
    return t


def _native(name, *args):
    """The extension's entry point: its result, or None where the call is not plain."""
    try:
        return getattr(_lib.torch_ext(), name)(*args)
    except RuntimeError as e:
        _lib.check_raised(e)


def _prepared(name, q, *args):
    """The same after the checks, with arguments that the kernels can read."""
    attention_error_word(q.device).poll()
    out = _native(name, q, *args)
    if out is None:
        raise _lib.NativeDeclined(f"{name} attention of {tuple(q.shape)} {q.dtype}")
    return out


def _as_mask(mask, device, shape, name):
    if mask.device != device:
        raise ValueError(f"{name} is on {mask.device}, q on {device}")
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(mask.shape)}")
    return mask if mask.dtype == torch.bool else mask != 0


def _attend(q, k, v, keep, scale, bias=None):
    """The formula in torch: q, k, v (..., length, dim) fp32, keep broadcastable to the scores."""
    s = (q @ k.transpose(-1, -2)) * scale
    if bias is not None:
        s = s + bias
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    top = s.detach().amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    return (p / torch.where(total == 0, torch.ones_like(total), total)) @ v


def _nothing(like, *inputs):
    """Zeros of `like`'s shape that depend on the inputs, whatever they hold."""
    return torch.zeros_like(like) + sum(t[:0].sum().to(like.dtype) for t in inputs)


# --------------------------------------------------------------------------- packed
def _ends(cu, device, name):
    if cu.dim() != 1 or cu.numel() < 1 or cu.dtype.is_floating_point or cu.dtype.is_complex or cu.dtype == torch.bool:
        raise ValueError(f"{name} must be a vector of whole numbers, got {cu.dtype} {tuple(cu.shape)}")
    if cu.device != device:
        raise ValueError(f"{name} is on {cu.device}, q on {device}")
    if cu.dtype not in (torch.int8, torch.uint8, torch.int16, torch.int32):   # past 32 bits: past any tensor, too
        cu = cu.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
    return cu.to(torch.int32).contiguous()


def _packed_torch(q, k, v, cu_q, cu_k, causal, scale, mask):
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    group = q.shape[1] // k.shape[1]
    pieces, at = [], 0
    for i in range(cu_q.numel() - 1):
        a, c = int(cu_q[i]), int(cu_k[i])
        b, d = int(cu_q[i + 1]), int(cu_k[i + 1])
        qs, n, m = q[a:b].float().transpose(0, 1), b - a, d - c
        keep = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            keep = keep.tril(m - n)
        if mask is not None:
            keep = keep & mask[c:d]
        rows = lambda t: (t[c:d].float() if mask is None else   # noqa: E731
                          t[c:d].float().masked_fill(~mask[c:d, None, None], 0)
                          ).transpose(0, 1).repeat_interleave(group, 0)
        if m == 0:
            o = _nothing(qs, qs, k, v)
        else:
            o = _attend(qs, rows(k), rows(v), keep, scale)
        pieces += [out[at:a], o.transpose(0, 1)]
        at = b
    return torch.cat([*pieces, out[at:]]).to(q.dtype)


def packed_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, *, causal=True, scale=None, key_mask=None):
    """Attention within each of B packed sequences.

    q: (rows, heads, dim); k, v: (rows, kv_heads, dim) with heads a multiple of kv_heads (query
    head h reads head h // (heads / kv_heads)). Sequence i is rows cu_seqlens[i] to
    cu_seqlens[i + 1] of q and the same rows of k and v, or cu_seqlens_k's: whole numbers on q's
    device that do not descend. Rows of no sequence give zeros. `causal`: query i of a sequence
    sees keys j <= i + (keys - queries), aligned to the last key, so a prompt's continuation
    passes its new queries and all keys. scale: dim ** -0.5 if None. key_mask: (rows of k,), keys
    with 0 / False are not seen and may hold anything (keys that only `causal` hides from some
    queries must be finite). Returns q's shape and type. Differentiable once in q, k and v."""
    if q.is_cuda and (cu_seqlens_k is not None or q.shape[0] == k.shape[0]):
        out = _native("packed", q, k, v, cu_seqlens, cu_seqlens if cu_seqlens_k is None else cu_seqlens_k,
                      bool(causal), scale, key_mask)
        if out is not None:
            return out
    if q.dim() != 3 or k.dim() != 3 or tuple(k.shape) != tuple(v.shape) or q.shape[2] != k.shape[2]:
        raise ValueError("packed_attention needs q (rows, heads, dim) and k, v (rows, kv_heads, dim), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    _heads(q.shape[1], k.shape[1], q.shape[2], q.is_cuda, q.dtype)
    _same(q.device, q.dtype, k=k, v=v)
    s = _scale(scale, q.shape[2])
    cu_q = _ends(cu_seqlens, q.device, "cu_seqlens")
    if cu_seqlens_k is None and q.shape[0] != k.shape[0]:
        raise ValueError("q and k have different numbers of rows: cu_seqlens_k is needed")
    cu_k = cu_q if cu_seqlens_k is None else _ends(cu_seqlens_k, q.device, "cu_seqlens_k")
    if cu_q.numel() != cu_k.numel():
        raise ValueError(f"{cu_q.numel() - 1} query sequences, {cu_k.numel() - 1} key sequences")
    mask = None if key_mask is None else _as_mask(key_mask, q.device, (k.shape[0],), "key_mask")
    if cu_q.numel() < 2 or q.shape[0] == 0 or k.shape[0] == 0:
        return _nothing(q, q, k, v)
    if not q.is_cuda:
        return _packed_torch(q, k, v, cu_q, cu_k, causal, s, mask)
    return _prepared("packed", _in_place(q), _in_place(k), _in_place(v), cu_q, cu_k, bool(causal), s,
                     None if mask is None else mask.contiguous())


# --------------------------------------------------------------------------- cached
def cached_attention(q, k_cache, v_cache, lengths, *, scale=None):
    """One new token of each sequence over its cache.

    q: (B, heads, dim); k_cache, v_cache: (B, capacity, kv_heads, dim), the new token's key and
    value included; lengths: (B,) whole numbers on q's device, how many positions of each cache
    hold keys (read on the device, clamped to 0 .. capacity: a captured graph replays with new
    lengths). A sequence of length 0 gives zeros. Returns (B, heads, dim). For inference: there is
    no backward, and inputs that want gradients are refused."""
    if q.is_cuda:
        out = _native("cached", q, k_cache, v_cache, lengths, scale)
        if out is not None:
            return out
    if q.dim() != 3 or k_cache.dim() != 4 or tuple(k_cache.shape) != tuple(v_cache.shape) or \
            q.shape[0] != k_cache.shape[0] or q.shape[2] != k_cache.shape[3]:
        raise ValueError("cached_attention needs q (B, heads, dim) and caches (B, capacity, kv_heads, dim), got "
                         f"{tuple(q.shape)}, {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    B, H, D = q.shape
    L, HK = k_cache.shape[1], k_cache.shape[2]
    _heads(H, HK, D, q.is_cuda, q.dtype)
    _same(q.device, q.dtype, k_cache=k_cache, v_cache=v_cache)
    s = _scale(scale, D)
    lens = _ends(lengths, q.device, "lengths") if B else lengths
    if tuple(lens.shape) != (B,):
        raise ValueError(f"lengths must have shape ({B},), got {tuple(lens.shape)}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_cache, v_cache)):
        raise ValueError("cached_attention has no backward: call it under torch.no_grad()")
    if B == 0 or L == 0:
        return torch.zeros_like(q)
    if not q.is_cuda:
        keep = torch.arange(L, device=q.device) < lens[:, None]
        rows = lambda t: t.float().masked_fill(~keep[..., None, None], 0).transpose(1, 2)   # noqa: E731
        o = _attend(q.float().view(B, HK, H // HK, D), rows(k_cache), rows(v_cache), keep[:, None, None], s)
        return o.reshape(B, H, D).to(q.dtype)
    return _prepared("cached", _in_place(q), _in_place(k_cache), _in_place(v_cache), lens, s)


# ----------------------------------------------------------------------------- pair
def pair_attention(q, k, v, bias, mask=None, *, scale=None):
    """Attention along the rows of a pair representation, with a bias that the rows share.

    q, k, v: (B, R, N, heads, dim) -- each of the B * R rows attends within itself; bias: (B or 1,
    heads, N, N), added to the scaled scores of every row, or None; mask: (B, R, N), keys with 0 /
    False are not seen (a row that has none left gives zeros). scale: dim ** -0.5 if None. Returns
    q's shape and type. Triangle attention has R = N; R = 1 is attention of a single representation
    with pair bias. Differentiable once in q, k, v and bias (its gradient summed over the rows)."""
    if q.is_cuda:
        out = _native("pair", q, k, v, bias, mask, scale)
        if out is not None:
            return out
    if q.dim() != 5 or tuple(k.shape) != tuple(q.shape) or tuple(v.shape) != tuple(q.shape):
        raise ValueError("pair_attention needs q, k and v of one shape (B, R, N, heads, dim), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, R, N, H, D = q.shape
    _heads(H, H, D, q.is_cuda, q.dtype)
    _same(q.device, q.dtype, k=k, v=v, bias=bias)
    s = _scale(scale, D)
    if bias is not None and (bias.dim() != 4 or bias.shape[0] not in (1, B) or tuple(bias.shape[1:]) != (H, N, N)):
        raise ValueError(f"bias must have shape ({B} or 1, {H}, {N}, {N}), got {tuple(bias.shape)}")
    m = None if mask is None else _as_mask(mask, q.device, (B, R, N), "mask")
    if q.numel() == 0:
        return _nothing(q, q, k, v, *(() if bias is None else (bias,)))
    if not q.is_cuda:
        keep = torch.ones(B, R, N, dtype=torch.bool, device=q.device) if m is None else m
        rows = lambda t: t.float().masked_fill(~keep[..., None, None], 0).transpose(2, 3)   # noqa: E731
        o = _attend(q.float().transpose(2, 3), rows(k), rows(v), keep[:, :, None, None, :], s,
                    None if bias is None else bias.float()[:, None])
        return o.transpose(2, 3).to(q.dtype)
    return _prepared("pair", _in_place(q), _in_place(k), _in_place(v), bias, None if m is None else m.contiguous(), s)
