"""GPU 3-bit KV cache and flash decode.

``Kv3Cache`` is one layer of the cache for ``batch`` sequences resident in
HBM (the C ABI's ``ft_kv3``): append, get_range, eviction and the split-S
flash decode over it.  ``TurboQuantKVCache`` keeps the reference's type and
call signatures (src/inference/turboquant_kv.rs:173-411: ``new``, ``append``,
``get_range``, ``get``, ``evict_oldest``, ``evict_to``, ``memory_bytes``,
``compression_ratio``, ``seq_len``, ``reset``) with one ``Kv3Cache`` per
layer, for a single sequence, host slices in and out.

The device cache stores exactly the reference's quantisation (group 128 = one
head vector: per-vector min and max, 3-bit codes), so ``export_range`` returns
the reference's stored bytes bit for bit.  Group sizes other than 128 raise
``UnsupportedError``.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from ._lib import ShapeError, UnsupportedError, call
from .gpu import _call_stream, _dptr, get_context

HEAD_DIM = 128
REC_BYTES = HEAD_DIM * 3 // 8  # 48
MAX_DRAFT = 64  # drafts of one tree: the bits of a mask word


def tree_mask(parents, device=None) -> torch.Tensor:
    """Ancestor masks of draft trees for ``tree_decode``: parents [..., n_draft] holds
    the index of each draft's parent (lower than its own), or -1 for a child of the
    prefix; bit j of mask[..., i] is set when draft j is i or an ancestor of i.
    Returns int64 masks on ``device`` (default: the current GPU)."""
    p = torch.as_tensor(parents).to(device="cpu", dtype=torch.int64)
    n = p.shape[-1] if p.dim() else 0
    if not 1 <= n <= MAX_DRAFT:
        raise ShapeError(f"a tree has 1 to {MAX_DRAFT} drafts")
    if bool(((p < -1) | (p >= torch.arange(n))).any()):
        raise ShapeError("a parent is -1 or the index of an earlier draft")
    m = torch.ones_like(p) << torch.arange(n)
    for _ in range(6):  # masks of the nearest 2^k ancestors, and the 2^k-th ancestor
        up = p.clamp(min=0)
        m = m | torch.where(p >= 0, m.gather(-1, up), 0)
        p = torch.where(p >= 0, p.gather(-1, up), -1)
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return m.to(device)


def _row_stride(t: torch.Tensor, rows: tuple, least: int, what: str, device) -> int:
    """Distance between the rows of an fp32 tensor [*rows, n >= least] on ``device``
    whose entries are adjacent and whose rows are equally spaced."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device or \
            t.dim() != 3 or tuple(t.shape[:2]) != tuple(rows) or t.shape[2] < least:
        raise ShapeError(f"{what} must be fp32 [{rows[0]}, {rows[1]}, >= {least}] on {device}")
    step = t.stride(1) if rows[1] > 1 else (t.stride(0) if rows[0] > 1 else t.shape[2])
    if (t.stride(2) != 1 and t.shape[2] > 1) or step < t.shape[2] or \
            (rows[0] > 1 and t.stride(0) != rows[1] * step):
        raise ShapeError(f"{what}: rows of adjacent entries, equally spaced, are expected")
    return step


def select_heavy(weights: torch.Tensor, n_keep: int, n_recent: int = 0, length: int | None = None,
                 seq_lens: torch.Tensor | None = None, stream=None):
    """The positions that an eviction by accumulated attention weight keeps.

    weights [batch, kv_heads, W] fp32 (``flash_decode(..., weights=...)``); of the first
    ``length`` (default W) or ``seq_lens[b]`` (int32 [batch] on the device) positions the
    ``n_recent`` last and the ``n_keep - n_recent`` heaviest of the others stay.  Returns
    (idx, weights): idx int32 [batch, kv_heads, n_keep], ascending, -1 where a sequence
    has fewer positions; a new weights tensor of the same shape with the kept
    positions' weights in front and zeros behind."""
    if not isinstance(weights, torch.Tensor) or weights.dim() != 3 or not weights.is_cuda:
        raise ShapeError("weights must be fp32 [batch, kv_heads, positions] on a GPU")
    B, H, W = weights.shape
    length = W if length is None else int(length)
    dev = weights.device
    if length < 0:
        raise ShapeError("a length is not negative")
    step = _row_stride(weights, (B, H), length, "weights", dev)
    if seq_lens is not None and (not isinstance(seq_lens, torch.Tensor) or
                                 seq_lens.dtype != torch.int32 or
                                 seq_lens.device != dev or tuple(seq_lens.shape) != (B,)):
        raise ShapeError(f"seq_lens must be int32 [{B}] on {dev}")
    n_keep, n_recent = int(n_keep), int(n_recent)
    if n_keep < 1 or not 0 <= n_recent <= n_keep:
        raise ShapeError("0 <= n_recent <= n_keep and n_keep >= 1 are expected")
    idx = weights.new_empty((B, H, n_keep), dtype=torch.int32)
    out = weights.new_empty((B, H, W))
    if B == 0 or W == 0:
        return idx.fill_(-1), out
    lens = None if seq_lens is None else seq_lens.contiguous()
    call("ft_kv_select_heavy", get_context(dev.index).handle, B, H, C.c_void_p(weights.data_ptr()),
         step, None if lens is None else _dptr(lens), length, n_keep, n_recent, _dptr(idx),
         _dptr(out), W, _call_stream(dev, stream, weights, idx, out, lens))
    return idx, out


def _index_list(idx: torch.Tensor, batch: int, kv_heads: int, device):
    """int32 index lists [n], [batch, n] or [batch, kv_heads, n] and their strides."""
    if not isinstance(idx, torch.Tensor) or idx.device != device or \
            idx.dtype not in (torch.int32, torch.int64):
        raise ShapeError(f"idx must be an int32 or int64 tensor on {device}")
    n = idx.shape[-1] if idx.dim() else 0
    if tuple(idx.shape) not in ((n,), (batch, n), (batch, kv_heads, n)) or idx.dim() == 0:
        raise ShapeError(f"idx must be [n], [{batch}, n] or [{batch}, {kv_heads}, n]")
    if idx.dtype == torch.int64:  # no wrap-around: what does not fit stays out of range
        idx = idx.clamp(-1, 2**31 - 1).to(torch.int32)
    idx = idx.contiguous()
    return idx, n, {1: (0, 0), 2: (n, 0), 3: (kv_heads * n, n)}[idx.dim()]


def _tree_args(q: torch.Tensor, mask, batch: int, device, out):
    """Checked q, mask and out of a tree decode: q [batch, n_draft, q_heads, 128]."""
    if not isinstance(q, torch.Tensor) or q.device != device or q.dim() != 4 or \
            q.dtype not in (torch.float32, torch.bfloat16) or q.shape[0] != batch or \
            q.shape[3] != HEAD_DIM:
        raise ShapeError(f"q must be fp32 or bf16 [{batch}, n_draft, q_heads, {HEAD_DIM}] "
                         f"on {device}")
    T = q.shape[1]
    if not 1 <= T <= MAX_DRAFT:
        raise UnsupportedError(f"{T} drafts: 1 to {MAX_DRAFT} are supported")
    q = q.contiguous()
    if q.data_ptr() % 16:  # a view that starts inside a row of its storage
        q = q.clone()
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.device != device or mask.dtype != torch.int64 \
                or mask.shape not in ((T,), (batch, T)):
            raise ShapeError(f"mask must be int64 [{T}] or [{batch}, {T}] on {device}")
        if mask.dim() == 1:
            mask = mask.expand(batch, T)
        mask = mask.contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or \
            out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ShapeError("out must be contiguous, 16-byte aligned and like q")
    return q, mask, out


def _decode_out(q: torch.Tensor, out) -> torch.Tensor:
    """The output of a single-token decode of ``q``: a new tensor, or ``out`` if it is
    contiguous and like q."""
    if out is None:
        return torch.empty_like(q)
    if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or \
            out.device != q.device or not out.is_contiguous():
        raise ShapeError("out must be contiguous and like q")
    return out


class Kv3Cache:
    """One layer's 3-bit KV cache for ``batch`` sequences on one GPU.

    ``stream``: a call runs there, behind what the current stream holds so far.  Calls on
    one cache share its scratch: they, and replays of graphs that hold them, follow one
    another."""

    def __init__(self, batch: int, kv_heads: int, max_seq: int, head_dim: int = HEAD_DIM,
                 device=None, mode: str = "R", seed: int = 0):
        """mode "R": the reference TurboQuantKVCache scheme (min/max per vector);
        mode "T": rotation + uniform 3-bit codebook + per-vector norm (see
        ft_kv3_create_mode), rotation signs drawn from ``seed``."""
        self.ctx = get_context(device)
        self.batch, self.kv_heads = int(batch), int(kv_heads)
        if mode not in ("R", "T"):
            raise ShapeError("mode must be 'R' or 'T'")
        self.mode = mode
        h = C.c_void_p()
        call("ft_kv3_create_mode", self.ctx.handle, self.batch, self.kv_heads, int(head_dim),
             int(max_seq), 0 if mode == "R" else 1, int(seed) & (2**64 - 1), C.byref(h))
        self.handle = h
        self.device = torch.device("cuda", self.ctx.device)

    def signs(self):
        """Mode T: the 128 rotation signs (numpy float32)."""
        import numpy as np
        out = np.empty(HEAD_DIM, np.float32)
        call("ft_kv3_signs", self.handle, out.ctypes.data_as(C.c_void_p))
        return out

    # ---- state
    def __len__(self) -> int:
        n = C.c_int64()
        call("ft_kv3_len", self.handle, C.byref(n))
        return n.value

    @property
    def capacity(self) -> int:
        n = C.c_int64()
        call("ft_kv3_capacity", self.handle, C.byref(n))
        return n.value

    def evict_front(self, n: int = 1) -> None:
        call("ft_kv3_evict_front", self.handle, int(n))

    def reset(self) -> None:
        call("ft_kv3_reset", self.handle)

    # ---- write
    def _kv_view(self, t: torch.Tensor) -> torch.Tensor:
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise ShapeError("K/V must be fp32 or bf16")
        t = t.contiguous()
        if t.numel() % (self.batch * self.kv_heads * HEAD_DIM):
            raise ShapeError("K/V must be [batch, n_pos, kv_heads, 128]")
        return t

    def append(self, k: torch.Tensor, v: torch.Tensor, stream=None) -> None:
        """k, v: [batch, n_pos, kv_heads, 128] (or [batch, n_pos, kv_dim]), fp32 or bf16."""
        k, v = self._kv_view(k), self._kv_view(v)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ShapeError("K and V must have the same shape and dtype")
        n = k.numel() // (self.batch * self.kv_heads * HEAD_DIM)
        call("ft_kv3_append", self.ctx.handle, self.handle, n, _dptr(k), _dptr(v),
             int(k.dtype == torch.bfloat16), _call_stream(self.device, stream, k, v))

    def append_packed(self, k_codes, k_minmax, v_codes, v_minmax, stream=None) -> None:
        """Positions in the reference's stored form: codes uint8 [batch, n, kv_heads*48],
        (min, max) fp32 [batch, n, kv_heads, 2]."""
        tens = [t.contiguous() for t in (k_codes, k_minmax, v_codes, v_minmax)]
        per = self.batch * self.kv_heads * REC_BYTES
        if tens[0].dtype != torch.uint8 or tens[0].numel() % per:
            raise ShapeError("codes must be uint8 [batch, n, kv_heads*48]")
        n = tens[0].numel() // per
        for t, w in ((tens[1], 2), (tens[3], 2)):
            if t.dtype != torch.float32 or t.numel() != self.batch * n * self.kv_heads * w:
                raise ShapeError("min/max must be fp32 [batch, n, kv_heads, 2]")
        if tens[2].shape != tens[0].shape or tens[2].dtype != torch.uint8:
            raise ShapeError("K and V codes must match")
        call("ft_kv3_append_packed", self.ctx.handle, self.handle, n, _dptr(tens[0]),
             _dptr(tens[1]), _dptr(tens[2]), _dptr(tens[3]),
             _call_stream(self.device, stream, *tens))

    # ---- read
    def get_range(self, start: int, end: int, stream=None):
        """Dequantised K, V [batch, end-start, kv_heads, 128] fp32 (reference get_range)."""
        n = int(end) - int(start)
        if n < 0:
            raise ShapeError("end < start")
        shape = (self.batch, n, self.kv_heads, HEAD_DIM)
        k = torch.empty(shape, dtype=torch.float32, device=self.device)
        v = torch.empty_like(k)
        call("ft_kv3_get_range", self.ctx.handle, self.handle, int(start), int(end), _dptr(k),
             _dptr(v), _call_stream(self.device, stream, k, v))
        return k, v

    def export_range(self, start: int, end: int, stream=None):
        """Reference stored form of positions [start, end): (k_codes, k_minmax, v_codes,
        v_minmax) with codes uint8 [batch, n, kv_heads*48] and min/max [batch, n, kv_heads, 2]."""
        n = int(end) - int(start)
        if n < 0:
            raise ShapeError("end < start")
        kc = torch.empty((self.batch, n, self.kv_heads * REC_BYTES), dtype=torch.uint8,
                         device=self.device)
        vc = torch.empty_like(kc)
        km = kc.new_empty((self.batch, n, self.kv_heads, 2), dtype=torch.float32)
        vm = torch.empty_like(km)
        call("ft_kv3_export_range", self.ctx.handle, self.handle, int(start), int(end),
             _dptr(kc), _dptr(km), _dptr(vc), _dptr(vm),
             _call_stream(self.device, stream, kc, km, vc, vm))
        return kc, km, vc, vm

    def flash_decode(self, q: torch.Tensor, scale: float = 0.0, out: torch.Tensor | None = None,
                     stream=None, weights: torch.Tensor | None = None) -> torch.Tensor:
        """q [batch, q_heads, 128] fp32 -> out [batch, q_heads, 128] fp32 over the whole
        cache; scale 0 selects 1/sqrt(128).  ``weights`` [batch, kv_heads, >= len] fp32:
        each position's attention weight, summed over the q heads of its kv head, is
        added to it (see ``evict_heavy``); the output is the same with and without."""
        if q.dtype != torch.float32 or q.dim() != 3 or q.shape[0] != self.batch or \
                q.shape[2] != HEAD_DIM:
            raise ShapeError("q must be fp32 [batch, q_heads, 128]")
        q = q.contiguous()
        out = _decode_out(q, out)
        if weights is not None:
            return self._decode_weights(q, scale, out, stream, weights)
        call("ft_flash_decode_3bit", self.ctx.handle, self.handle, _dptr(q), int(q.shape[1]),
             float(scale), _dptr(out), _call_stream(self.device, stream, q, out))
        return out

    def _decode_weights(self, q, scale, out, stream, weights):
        if q.device != self.device:
            raise ShapeError(f"q must be on {self.device}")
        step = _row_stride(weights, (self.batch, self.kv_heads), len(self), "weights", self.device)
        call("ft_flash_decode_3bit_weights", self.ctx.handle, self.handle, _dptr(q),
             int(q.shape[1]), float(scale), _dptr(out), C.c_void_p(weights.data_ptr()), step,
             _call_stream(self.device, stream, q, out, weights))
        return out

    def tree_decode(self, q: torch.Tensor, mask: torch.Tensor | None = None, scale: float = 0.0,
                    out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Attention of drafted tokens: the last n_draft (1..64) positions of the cache are
        the drafts (append them first).  q [batch, n_draft, q_heads, 128] fp32 or bf16 ->
        out of the same type; draft i sees all earlier positions and the drafts named by
        the bits of mask[b, i] (int64 [batch, n_draft] or [n_draft], see ``tree_mask``;
        None: drafts 0..i).  A draft that sees nothing gets 0."""
        q, mask, out = _tree_args(q, mask, self.batch, self.device, out)
        call("ft_kv3_tree_decode", self.ctx.handle, self.handle, int(q.shape[1]), _dptr(q),
             int(q.dtype == torch.bfloat16), int(q.shape[2]), None if mask is None else _dptr(mask),
             float(scale), _dptr(out), _call_stream(self.device, stream, q, out, mask))
        return out

    # ---- choosing what stays
    def keep(self, idx: torch.Tensor, start: int = 0, stream=None) -> None:
        """Positions below ``start`` and the listed ones stay, the rest is dropped: new
        position start + i is old position idx[..., i] for each sequence and kv head
        (idx [n], [batch, n] or [batch, kv_heads, n], ascending from ``start`` on).  After
        a tree decode: the accepted path.  An entry outside [start + i, len) is skipped
        and reported by ``ctx.check()``.  (A ring that is full from the middle of a block
        on may be laid out anew, as by an append that grows it: graphs captured before
        then no longer hold.)"""
        idx, n, (ib, ih) = _index_list(idx, self.batch, self.kv_heads, self.device)
        self._keep(idx, n, ib, ih, int(start), stream)

    def _keep(self, idx, n, ib, ih, start, stream):
        call("ft_kv3_keep", self.ctx.handle, self.handle, start, n, _dptr(idx), ib, ih,
             _call_stream(self.device, stream, idx))

    def evict_heavy(self, weights: torch.Tensor, n_keep: int, n_recent: int = 0, stream=None):
        """Evicts down to ``n_keep`` positions per sequence and kv head: the ``n_recent``
        last and the heaviest of the others by accumulated attention ``weights``
        [batch, kv_heads, >= len] stay (``select_heavy``).  Returns (idx, weights): the
        kept old positions and the weights that belong to the new ones."""
        n = len(self)
        if not isinstance(weights, torch.Tensor) or weights.device != self.device or \
                tuple(weights.shape[:2]) != (self.batch, self.kv_heads):
            raise ShapeError(f"weights must be fp32 [{self.batch}, {self.kv_heads}, >= {n}] "
                             f"on {self.device}")
        idx, out = select_heavy(weights, n_keep, n_recent, length=n, stream=stream)
        if n > int(n_keep):
            self._keep(idx, int(n_keep), self.kv_heads * int(n_keep), int(n_keep), 0, stream)
        return idx, out

    def close(self):
        if getattr(self, "handle", None):
            call("ft_kv3_destroy", self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class TurboQuantKVCache:
    """The reference's ``TurboQuantKVCache`` (turboquant_kv.rs:173-411) for one
    sequence, one ``Kv3Cache`` per layer in HBM."""

    def __init__(self, num_layers: int, kv_dim: int, max_seq_len: int, group_size: int,
                 device=None):
        if group_size != HEAD_DIM or kv_dim % HEAD_DIM or kv_dim <= 0:
            raise UnsupportedError(
                "the device cache quantises one 128-value head vector per group: group_size "
                "must be 128 and kv_dim a multiple of 128")
        self.num_layers = int(num_layers)
        self.kv_dim = int(kv_dim)
        self.group_size = int(group_size)
        self.max_seq_len = int(max_seq_len)
        self.num_groups = (kv_dim + group_size - 1) // group_size
        self.bytes_per_pos = (kv_dim * 3 + 7) // 8
        self.current_len = 0
        self.layers = [Kv3Cache(1, kv_dim // HEAD_DIM, max(1, max_seq_len), device=device)
                       for _ in range(self.num_layers)]
        self.device = self.layers[0].device

    def _vec(self, a) -> torch.Tensor:
        t = a if isinstance(a, torch.Tensor) else torch.from_numpy(
            np.ascontiguousarray(np.asarray(a, dtype=np.float32)))
        if t.numel() != self.kv_dim:
            raise ShapeError(f"expected a vector of kv_dim = {self.kv_dim} values")
        if t.dtype not in (torch.float32, torch.bfloat16):
            t = t.float()
        return t.to(self.device).reshape(1, 1, self.kv_dim)

    def append(self, layer: int, k, v) -> None:
        """append (:240-266): quantise and store one position of ``layer``."""
        self.layers[layer].append(self._vec(k), self._vec(v))
        if layer == self.num_layers - 1:
            self.current_len += 1

    def get_range(self, layer: int, start: int, end: int):
        """get_range (:271-291): (K, V) as flat fp32 host arrays of (end-start)*kv_dim;
        positions past the layer's stored length are zeros."""
        if end < start:
            raise ShapeError("end < start")
        n = end - start
        k = np.zeros(n * self.kv_dim, np.float32)
        v = np.zeros(n * self.kv_dim, np.float32)
        have = min(end, len(self.layers[layer])) - start
        if have > 0:
            kd, vd = self.layers[layer].get_range(start, start + have)
            k[:have * self.kv_dim] = kd.reshape(-1).cpu().numpy()
            v[:have * self.kv_dim] = vd.reshape(-1).cpu().numpy()
        return k, v

    def get(self, layer: int, pos: int):
        """get (:294-305)."""
        return self.get_range(layer, pos, pos + 1)

    def evict_oldest(self) -> None:
        """evict_oldest (:308-320)."""
        for c in self.layers:
            if len(c):
                c.evict_front(1)
        if self.current_len > 0:
            self.current_len -= 1

    def evict_to(self, target_len: int) -> None:
        """evict_to (:323-327)."""
        while self.current_len > target_len:
            self.evict_oldest()

    def memory_bytes(self) -> int:
        """memory_bytes (:330-336): the reference's per-position accounting."""
        per_pos = self.bytes_per_pos * 2 + self.num_groups * 2 * 4 * 2
        return per_pos * self.current_len * self.num_layers

    def compression_ratio(self) -> float:
        """compression_ratio (:338-343)."""
        fp32_per_pos = self.kv_dim * 4 * 2
        denom = self.current_len * self.num_layers
        actual = self.memory_bytes() / denom if denom else float("nan")
        return fp32_per_pos / actual if actual > 0 else 1.0

    def seq_len(self) -> int:
        return self.current_len

    def reset(self) -> None:
        for c in self.layers:
            c.reset()
        self.current_len = 0

    def flash_decode(self, layer: int, q, q_heads: int, scale: float = 0.0) -> np.ndarray:
        """Attention of q [q_heads * 128] over the layer's cache (flash_decode_ref math
        with the GQA head map); host in, host out."""
        qt = q if isinstance(q, torch.Tensor) else torch.from_numpy(
            np.ascontiguousarray(np.asarray(q, dtype=np.float32)))
        qt = qt.float().to(self.device).reshape(1, q_heads, HEAD_DIM)
        return self.layers[layer].flash_decode(qt, scale).reshape(-1).cpu().numpy()

    def close(self):
        for c in self.layers:
            c.close()
