"""The attention half of a block served from an 8-bit cache: rotary positions,
the paged cache (write, read back) and attention over it.

Torch tensors in and out over the C ABI's noor_rope_apply, noor_kv_append,
noor_kv_read and noor_kv_attention (include/noor_moe.h states what each
computes).  Every call runs on the tensors' device and on that device's
current torch stream, allocates only through torch (so it can be captured into
a CUDA graph) and never synchronises.  The reference's counterparts are
RoPE::apply (crates/noor-core/src/layers/rope.rs:49-90) and
GQAAttention::forward with its KV cache (attention.rs:67-191).

There is no CPU fallback: tensors must be on a CUDA device.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Sequence, Tuple, Union

import numpy as np

from . import api

LAYOUTS = {"interleaved": 0, "half": 1}
FORMATS = {"int8": 0, "e4m3": 1}
STATUS = {1: "row offsets are not ascending within the rows given",
          2: "a length is negative, below the sequence's rows, or past its pages",
          3: "a page number is outside the cache",
          4: "a bounded wait on the device gave up"}


# A decode step's calls cost more on the host than on the GPU, so arguments are
# packed as the C structures' bytes (noor_heads, noor_kv_batch) and each tensor
# is asked for its shape and strides once.
_HEADS = struct.Struct("Pqq")
_BATCH = struct.Struct("PqPPqii")


_T = None


def _torch():
    global _T
    if _T is None:
        import torch
        _T = torch
    return _T


def _code_dtype(fmt: str):
    torch = _torch()
    return torch.int8 if fmt == "int8" else torch.float8_e4m3fn


def _dtype_code(t) -> int:
    torch = _torch()
    if t.dtype is torch.bfloat16:
        return api.DTYPE_BF16
    if t.dtype is torch.float32:
        return api.DTYPE_F32
    raise ValueError(f"expected bfloat16 or float32, got {t.dtype}")


def _heads(t, what: str, device: int, dim: int) -> bytes:
    """noor_heads of a tensor [tokens, heads, dim] on CUDA device `device`."""
    st = t.stride()
    if len(st) != 3 or t.get_device() != device:
        raise ValueError(f"{what} must be a tensor [tokens, heads, head_dim] on cuda:{device}, got {tuple(t.shape)} on "
                         f"{t.device}")
    if t.size(2) != dim:
        raise ValueError(f"{what} has head_dim {t.size(2)}, expected {dim}")
    if st[2] != 1 and dim > 1:
        raise ValueError(f"{what}: a head's elements must be contiguous")
    return _HEADS.pack(t.data_ptr(), st[0], st[1])


def _ints(t, what: str, n: int, device: int) -> int:
    """Data pointer of a contiguous int32 tensor [n] on `device`."""
    st = t.stride()
    if t.dtype is not _T.int32 or t.get_device() != device or len(st) != 1 or t.size(0) != n or (st[0] != 1 and n > 1):
        raise ValueError(f"{what} must be a contiguous int32 tensor ({n},) on cuda:{device}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t.data_ptr()


def _tangent(t):
    """t's forward-mode tangent, None without one (and outside of dual levels, at
    once)."""
    fw = _T.autograd.forward_ad
    if t is None or getattr(fw, "_current_level", 0) < 0:
        return None
    return fw.unpack_dual(t).tangent


def _no_grad(*tensors) -> None:
    """The cache rounds to 8 bits and holds no graph: refuse what wants a gradient
    or carries a tangent."""
    grad = _T.is_grad_enabled()
    for t in tensors:
        if t is not None and (grad and t.requires_grad or _tangent(t) is not None):
            raise ValueError("the cached path has no gradient: call it under torch.no_grad() or detach its inputs, without "
                             "forward-mode tangents")


def _empty_like(t):
    """Contiguous output of t's shape."""
    return _T.empty_like(t, memory_format=_T.contiguous_format)


def _stream(device: int) -> int:
    return _torch()._C._cuda_getCurrentRawStream(device)


# ------------------------------------------------------------ rotary


def rotary_frequencies(head_dim: int, theta: float = 10000.0, fraction: Optional[float] = None, *,
                       linear: float = 1.0, ntk: float = 1.0,
                       yarn: Optional[dict] = None) -> Tuple[np.ndarray, float]:
    """Inverse frequencies (f32) of the rotated pairs and the attention factor.

    theta and fraction as RoPE::new / new_proportional (rope.rs:17-45).  For
    contexts longer than the trained one, at most one of
      linear  s: positions are divided by s;
      ntk     s: theta grows by s^(rot / (rot - 2)), which leaves the fastest
              pair as it is and divides the slowest by s;
      yarn    {"scale": s, "original": trained context, "fast": 32, "slow": 1}:
              pairs that turn more than `fast` times over the trained context
              keep their frequency, those below `slow` turns are divided by s,
              a linear ramp between (Peng et al., "YaRN", 2023); the factor is
              0.1 ln s + 1.
    """
    rot = head_dim if fraction is None else max(2, (int(head_dim * fraction) // 2) * 2)
    if rot > head_dim or rot % 2:
        raise ValueError(f"cannot rotate {rot} of {head_dim} dims")
    if sum((linear != 1.0, ntk != 1.0, yarn is not None)) > 1:
        raise ValueError("at most one of linear, ntk and yarn")
    for what, x in (("theta", theta), ("linear", linear), ("ntk", ntk), *(() if yarn is None else (
            ("yarn's scale", yarn["scale"]), ("yarn's original", yarn["original"])))):
        if not (0 < x < math.inf):
            raise ValueError(f"{what} must be positive and finite, got {x}")
    if ntk != 1.0 and rot > 2:
        theta = theta * ntk ** (rot / (rot - 2.0))
    inv = theta ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot) / linear
    factor = 1.0
    if yarn is not None:
        s = float(yarn["scale"])
        fast, slow = float(yarn.get("fast", 32.0)), float(yarn.get("slow", 1.0))
        if not (-math.inf < slow < fast < math.inf):
            raise ValueError(f"yarn's fast must be above its slow, got {fast} and {slow}")
        turns = float(yarn["original"]) * inv / (2.0 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        inv = inv / s * (1.0 - keep) + inv * keep
        factor = 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
    return inv.astype(np.float32), factor


class Rotary:
    """A table of inverse frequencies on a device, its layout and factor.

    inv_freq: f32 tensor (or numpy array, uploaded to `device`) of rotate_dim / 2
    frequencies; layout "interleaved" (pairs 2i, 2i + 1, the reference's) or
    "half" (pairs i, i + rotate_dim / 2)."""

    def __init__(self, inv_freq, layout: str = "interleaved", factor: float = 1.0, device: Union[int, str] = 0):
        torch = _torch()
        if layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}")
        if isinstance(inv_freq, np.ndarray):
            inv_freq = torch.from_numpy(np.ascontiguousarray(inv_freq, np.float32)).to(torch.device("cuda", device) if isinstance(
                device, int) else device)
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_cuda:
            raise ValueError("inv_freq must be a 1-D float32 CUDA tensor")
        if inv_freq.requires_grad or _tangent(inv_freq) is not None:
            raise ValueError("the frequencies have no gradient: detach them")
        self.inv_freq = inv_freq.contiguous()
        self.rotate_dim = 2 * inv_freq.numel()
        self.layout, self.factor = layout, float(factor)
        self.device = self.inv_freq.get_device()
        self.desc = api.RotaryDesc(self.inv_freq.data_ptr(), self.rotate_dim, LAYOUTS[layout], self.factor)
        self.ref = ctypes.byref(self.desc)

    @classmethod
    def create(cls, head_dim: int, theta: float = 10000.0, fraction: Optional[float] = None,
               layout: str = "interleaved", device: Union[int, str] = 0, **scaling) -> "Rotary":
        inv, factor = rotary_frequencies(head_dim, theta, fraction, **scaling)
        return cls(inv, layout, factor, device)


def _rope_call(q, k, positions, rotary: Rotary, inverse: bool):
    torch = _torch()
    dt = _dtype_code(q)
    if q.dim() != 3 or not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor [tokens, heads, head_dim], got {tuple(q.shape)} on {q.device}")
    T, nq, D = q.shape
    dev = q.get_device()
    hq = _heads(q, "q", dev, D)
    if rotary.device != dev:
        raise ValueError(f"the rotary table is on cuda:{rotary.device}, q on cuda:{dev}")
    pos = _ints(positions, "positions", T, dev)
    q_out = _empty_like(q)
    k_out = hk = hk_out = None
    nk = 0
    if k is not None:
        hk = _heads(k, "k", dev, D)
        nk = k.size(1)
        if k.dtype is not q.dtype or k.size(0) != T:
            raise ValueError("k must have q's tokens and type")
        k_out = _empty_like(k)
        hk_out = _HEADS.pack(k_out.data_ptr(), nk * D, D)
    rc = api.lib().noor_rope_apply(rotary.ref, hq, _HEADS.pack(q_out.data_ptr(), nq * D, D), nq, hk, hk_out, nk, pos, T, D,
                                   dt, inverse, dev, _stream(dev))
    if rc:
        api.check(rc)
    return q_out, k_out


_rope_function = None


def _rope_autograd():
    """The autograd function, made on first use (torch is imported lazily)."""
    global _rope_function
    if _rope_function is None:
        torch = _torch()

        class RopeFunction(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, positions, rotary, inverse):
                ctx.args = (rotary, inverse)
                ctx.set_materialize_grads(False)
                ctx.save_for_backward(positions)
                q_out, k_out = _rope_call(q, k, positions, rotary, inverse)
                return q_out if k is None else (q_out, k_out)

            @staticmethod
            def backward(ctx, gq, gk=None):
                # The transpose: the rotation the other way, itself differentiable.
                # Gradients may come broadcast, or not at all.
                rotary, inverse = ctx.args
                (positions,) = ctx.saved_tensors
                need = ctx.needs_input_grad
                gq = gq if need[0] else None
                gk = gk if need[1] else None
                if gq is not None and gq.stride(-1) != 1:
                    gq = gq.contiguous()
                if gk is not None and gk.stride(-1) != 1:
                    gk = gk.contiguous()
                if gq is None and gk is None:
                    return None, None, None, None, None
                first, second = (gq, gk) if gq is not None else (gk, None)
                d0, d1 = _rope(first, second, positions, rotary, not inverse)
                return (d0, d1, None, None, None) if gq is not None else (None, d0, None, None, None)

        _rope_function = RopeFunction
    return _rope_function


def _rope(q, k, positions, rotary: Rotary, inverse: bool):
    """(q', k') of q and k (or None), with their derivatives where asked for."""
    torch = _torch()
    tq, tk = _tangent(q), _tangent(k)
    if tq is not None or tk is not None:  # linear in q and k: tangents turn alike
        fw = torch.autograd.forward_ad
        out = list(_rope(fw.unpack_dual(q).primal, None if k is None else fw.unpack_dual(k).primal, positions, rotary, inverse))
        for i, t in enumerate((tq, tk)):
            if t is not None:
                t = t if t.stride(-1) == 1 else t.contiguous()
                out[i] = fw.make_dual(out[i], _rope(t, None, positions, rotary, inverse)[0])
        return tuple(out)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _rope_autograd().apply(q, k, positions, rotary, inverse)
        return (out, None) if k is None else out
    return _rope_call(q, k, positions, rotary, inverse)


def rope_apply(q, positions, rotary: Rotary, k=None):
    """Rotate q [tokens, heads, head_dim] (and k beside it, in one launch) to
    positions [tokens] (int32).  Differentiable in q and k, backward and forward;
    returns new tensors q', or (q', k')."""
    q_out, k_out = _rope(q, k, positions, rotary, False)
    return q_out if k is None else (q_out, k_out)


# ------------------------------------------------------------ cache


class KVCache:
    """A paged cache of keys and values in 8 bits (noor_kv_cache).

    A page holds `block` tokens of every kv head; k_codes [pages, kv heads,
    block, head_dim], v_codes [pages, kv heads, head_dim, block], int8 or
    float8_e4m3fn; k_scale and v_scale [pages, kv heads] f32.  The caller owns
    the pages: block_table [batch, max_blocks] int32 names those of each
    sequence, kv_lens [batch] int32 its tokens (a call's new ones included),
    cu_rows [batch + 1] int32 the rows of each sequence in the row tensors;
    all three stay on the device, so one captured graph serves changing
    lengths.  Mistakes in them never reach memory outside the buffers: the
    rows concerned are skipped or come back NaN, and check() raises."""

    def __init__(self, num_blocks: int, n_kv_heads: int, head_dim: int, block: int = 64, fmt: str = "int8",
                 device: int = 0):
        torch = _torch()
        if fmt not in FORMATS:
            raise ValueError(f"unknown cache format {fmt!r}")
        dev = torch.device("cuda", device)
        z = lambda shape: torch.zeros(shape, dtype=torch.int8, device=dev).view(_code_dtype(fmt))
        self._bind(z((num_blocks, n_kv_heads, block, head_dim)), z((num_blocks, n_kv_heads, head_dim, block)),
                   torch.zeros((num_blocks, n_kv_heads), device=dev), torch.zeros((num_blocks, n_kv_heads), device=dev))

    @classmethod
    def from_tensors(cls, k_codes, v_codes, k_scale, v_scale) -> "KVCache":
        """A cache over tensors the caller holds (kept, not copied)."""
        c = cls.__new__(cls)
        c._bind(k_codes, v_codes, k_scale, v_scale)
        return c

    def _bind(self, k_codes, v_codes, k_scale, v_scale) -> None:
        torch = _torch()
        if k_codes.dim() != 4 or not k_codes.is_cuda:
            raise ValueError("k_codes must be a CUDA tensor [pages, kv heads, block, head_dim]")
        P, H, blk, D = k_codes.shape
        fmt = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}.get(k_codes.dtype)
        if fmt is None or v_codes.dtype != k_codes.dtype:
            raise ValueError(f"codes must both be int8 or float8_e4m3fn, got {k_codes.dtype} and {v_codes.dtype}")
        for name, t, shape in (("v_codes", v_codes, (P, H, D, blk)), ("k_scale", k_scale, (P, H)),
                               ("v_scale", v_scale, (P, H))):
            if tuple(t.shape) != shape or t.device != k_codes.device:
                raise ValueError(f"{name} must have shape {shape} on {k_codes.device}")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes), ("k_scale", k_scale), ("v_scale", v_scale)):
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if name.endswith("scale") and t.dtype != torch.float32:
                raise ValueError(f"{name} must be float32")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.num_blocks, self.n_kv_heads, self.block, self.head_dim = P, H, blk, D
        self.format, self.device = fmt, k_codes.device
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._dev = k_codes.get_device()
        self.desc = api.KVCacheDesc(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                    self.status.data_ptr(), P, H, D, blk, FORMATS[fmt], self._dev)
        self._ref = ctypes.byref(self.desc)
        self._workspace = {}  # bytes of attention's workspace by its sizes

    def check(self) -> None:
        """Wait for the device (every stream's calls) and raise NoorMoEError if a
        kernel found a mistake in device metadata since the last check; clears it."""
        _torch().cuda.synchronize(self.device)
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise api.NoorMoEError(6 if code == 4 else 1, f"cache: {STATUS.get(code, code)}")

    def _batch(self, block_table, kv_lens, cu_rows, rows: int) -> bytes:
        """noor_kv_batch."""
        if block_table.dim() != 2 or block_table.dtype is not _torch().int32 or block_table.get_device() != self._dev:
            raise ValueError(f"block_table must be an int32 tensor [batch, max_blocks] on cuda:{self._dev}, got "
                             f"{block_table.dtype} {tuple(block_table.shape)} on {block_table.device}")
        B, maxb = block_table.shape
        ts = block_table.stride()
        if ts[1] != 1 and maxb > 1:
            raise ValueError("block_table's rows must be contiguous")
        return _BATCH.pack(block_table.data_ptr(), ts[0],
                           0 if kv_lens is None else _ints(kv_lens, "kv_lens", B, self._dev),
                           _ints(cu_rows, "cu_rows", B + 1, self._dev), rows, B, maxb)

    def append(self, k, v, block_table, kv_lens, cu_rows, rotary: Optional[Rotary] = None, q=None):
        """Write the new tokens' k and v [rows, kv heads, head_dim]; row i of
        sequence b is its token kv_lens[b] - rows(b) + i.  With `rotary`, keys
        are rotated to their positions first, and q [rows, heads, head_dim]
        beside them: the rotated q is returned (rows past the last sequence's are
        undefined), else None."""
        torch = _torch()
        dt = _dtype_code(k)
        dev, D = self._dev, self.head_dim
        hk, hv = _heads(k, "k", dev, D), _heads(v, "v", dev, D)
        _no_grad(k, v, q)
        rows = k.size(0)
        if k.size(1) != self.n_kv_heads or v.size(1) != self.n_kv_heads:
            raise ValueError(f"k and v must have {self.n_kv_heads} heads")
        if v.size(0) != rows or v.dtype is not k.dtype:
            raise ValueError("v must have k's rows and type")
        batch = self._batch(block_table, kv_lens, cu_rows, rows)
        rot = q_out = hq = hq_out = None
        nq = 0
        if rotary is not None:
            if rotary.device != dev:
                raise ValueError(f"the rotary table is on cuda:{rotary.device}, the cache on cuda:{dev}")
            rot = rotary.ref
        if q is not None:
            if rotary is None:
                raise ValueError("q is rotated beside the write: it needs `rotary`")
            hq = _heads(q, "q", dev, D)
            nq = q.size(1)
            if q.size(0) != rows or q.dtype is not k.dtype:
                raise ValueError("q must have k's rows and type")
            q_out = _empty_like(q)
            hq_out = _HEADS.pack(q_out.data_ptr(), nq * D, D)
        rc = api.lib().noor_kv_append(self._ref, batch, hk, hv, rot, hq, hq_out, nq, dt, _stream(dev))
        if rc:
            api.check(rc)
        return q_out

    def read(self, block_table, starts, cu_rows, rows: int, dtype=None, kv_lens=None):
        """Tokens read back: row i of sequence b is its token starts[b] + i
        (starts None: from 0).  rows: rows of the result, at least cu_rows[-1].
        kv_lens bounds the tokens (None: the tables' whole width).  Returns k, v
        [rows, kv heads, head_dim] in `dtype` (bfloat16 by default)."""
        torch = _torch()
        batch = self._batch(block_table, kv_lens, cu_rows, rows)
        st = None if starts is None else _ints(starts, "starts", block_table.size(0), self._dev)
        shape = (rows, self.n_kv_heads, self.head_dim)
        dtype = torch.bfloat16 if dtype is None else dtype
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        rc = api.lib().noor_kv_read(self._ref, batch, st, k.data_ptr(), v.data_ptr(), _dtype_code(k), _stream(self._dev))
        if rc:
            api.check(rc)
        return k, v

    def attention(self, q, block_table, kv_lens, cu_rows, max_rows: int, scale: Optional[float] = None,
                  window: int = 0, out=None, return_lse: bool = False):
        """Causal attention of q [rows, heads, head_dim] over the cache: row i
        of sequence b is at position kv_lens[b] - rows(b) + i.  max_rows: the
        most rows of a sequence (a hint).  window > 0: keys at most `window`
        positions back.  scale: 1 / sqrt(head_dim) by default.  Returns out, or
        (out, lse) with lse [rows, heads] f32.  `out` may be q."""
        torch = _torch()
        dt = _dtype_code(q)
        dev, D = self._dev, self.head_dim
        hq = _heads(q, "q", dev, D)
        _no_grad(q, out)
        rows, nq = q.size(0), q.size(1)
        if nq % self.n_kv_heads != 0:
            raise ValueError(f"{nq} query heads over {self.n_kv_heads} kv heads")
        batch = self._batch(block_table, kv_lens, cu_rows, rows)
        if out is None:
            out = _empty_like(q)
            ho = _HEADS.pack(out.data_ptr(), nq * D, D)
        else:
            if out.shape != q.shape or out.dtype is not q.dtype:
                raise ValueError("out must have q's shape and type")
            ho = _heads(out, "out", dev, D)
        lse = torch.empty((rows, nq), dtype=torch.float32, device=q.device) if return_lse else None
        lib = api.lib()
        key = (rows, nq, max_rows, dt, *block_table.shape)
        need = self._workspace.get(key)
        if need is None:
            n = ctypes.c_int64()
            api.check(lib.noor_kv_attention_workspace(self._ref, batch, nq, max_rows, dt, ctypes.byref(n)))
            if len(self._workspace) >= 1024:  # a server's prompts come in any number of rows
                self._workspace.clear()
            need = self._workspace[key] = n.value
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        rc = lib.noor_kv_attention(self._ref, batch, hq, ho, lse.data_ptr() if return_lse else None, nq, max_rows,
                                   D ** -0.5 if scale is None else scale, min(window, 2 ** 31 - 1), dt, ws.data_ptr(), need, _stream(dev))
        if rc:
            api.check(rc)
        return (out, lse) if return_lse else out
