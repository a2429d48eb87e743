"""Host-side API of the latent-cache attention operators (include/loki_attn.h): rotary positions, the paged latent
cache, attention of drafted token trees over it, the attention weight of each cached row, and eviction by it.

The cache holds the row that the reference's attention keeps (latent 512, rotated key part 64; src/fused_layer.cu:277-308);
torch supplies device memory and streams, every computation runs in libloki_moe.so.  Calls are queued on the current
stream (or `stream`) and do not synchronise; AttnContext.device_error() reports what a kernel refused.
"""
import ctypes

import torch

from . import native as N
from .moe import _ptr, _stream
from .native import ATTN_LATENT, ATTN_ROPE, ATTN_ROW, check, lib

_DTYPE = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}
_LAYOUT = {"interleaved": N.ROPE_INTERLEAVED, "half": N.ROPE_HALF}


def _need(cond, msg, *args):
    if not cond:
        raise ValueError(msg % args if args else msg)


def _dense(t, name, dtype, device, *shape):
    """A contiguous tensor of this dtype and shape (None: any size) on the device."""
    _need(isinstance(t, torch.Tensor) and t.device == device and t.dtype in dtype and t.is_contiguous(),
          "%s: a contiguous %s tensor on %s", name, "/".join(str(d) for d in dtype), device)
    _need(t.dim() == len(shape) and all(s is None or s == n for s, n in zip(shape, t.shape)), "%s: shape %s, wanted %s",
          name, tuple(t.shape), shape)
    return t


def _rows(t, name, device, last, dim):
    """A tensor whose last dimension is `last` wide and dense; the other strides are free."""
    _need(isinstance(t, torch.Tensor) and t.device == device and t.dim() == dim and (last is None or t.shape[-1] == last) and
          (t.shape[-1] <= 1 or t.stride(-1) == 1), "%s: a %d-d tensor on %s with a dense last dimension%s", name, dim, device,
          "" if last is None else " of %d" % last)
    return t


class RopeTable:
    """cos and sin of positions 0 .. max_pos-1 ([max_pos][rot_dim / 2][2] fp32), angles in 64 bits.  factor > 1 stretches
    the context: frequencies of fewer than beta_slow turns over orig_ctx are divided by factor, those of more than
    beta_fast are kept, with a linear mix between; cos and sin are multiplied by mscale."""

    def __init__(self, max_pos, rot_dim=ATTN_ROPE, base=10000.0, factor=1.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0,
                 mscale=1.0, device="cuda", stream=None):
        device = torch.device(device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.max_pos, self.rot_dim = max_pos, rot_dim
        self.table = torch.empty(max(max_pos, 0), max(rot_dim, 0) // 2, 2, device=device)
        cfg = N.LkRopeConfig(rot_dim, base, factor, orig_ctx, beta_fast, beta_slow, mscale)
        with torch.cuda.device(device):
            check(lib().lk_attn_rope_table(None, ctypes.byref(cfg), max_pos, _ptr(self.table), _stream(stream)))


class KvCache:
    """The paged latent cache of n_seqs sequences over caller-owned tensors.

    rows [n_pages * page_size][576] fp16 or bf16 (a row stride above 576 is fine); block_table [n_seqs][pages] int32;
    lens [n_seqs] int32, rows of context; mass fp32 and pos int32 [n_pages * page_size], optional (eviction needs both)."""

    def __init__(self, rows, page_size, block_table, lens, mass=None, pos=None):
        dev = rows.device
        _rows(rows, "rows", dev, ATTN_ROW, 2)
        _need(rows.dtype in (torch.float16, torch.bfloat16), "rows: fp16 or bf16")
        _need(page_size >= 1 and rows.shape[0] % page_size == 0, "rows: %d is not a multiple of the page size %d", rows.shape[0], page_size)
        _dense(block_table, "block_table", (torch.int32,), dev, None, None)
        _dense(lens, "lens", (torch.int32,), dev, block_table.shape[0])
        if mass is not None:
            _dense(mass, "mass", (torch.float32,), dev, rows.shape[0])
        if pos is not None:
            _dense(pos, "pos", (torch.int32,), dev, rows.shape[0])
        self.rows, self.page_size, self.block_table, self.lens, self.mass, self.pos = rows, page_size, block_table, lens, mass, pos
        self.device = dev
        self.n_seqs = block_table.shape[0]
        self._struct = N.LkKvCache(rows.data_ptr(), rows.stride(0), _DTYPE[rows.dtype], page_size, rows.shape[0] // page_size,
                                   block_table.data_ptr(), block_table.shape[1], self.n_seqs, lens.data_ptr(),
                                   None if mass is None else mass.data_ptr(), None if pos is None else pos.data_ptr())

    def struct(self):
        return ctypes.byref(self._struct)


class AttnContext:
    """Workspaces of the attention operators for up to max_seqs sequences and max_tokens drafted tokens per call, on one
    device.  Calls on one context run on one stream at a time."""

    def __init__(self, device=0, max_seqs=64, max_tokens=512):
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        cfg = N.LkAttnConfig(max_seqs, max_tokens)
        h = ctypes.c_void_p()
        check(lib().lk_attn_create(ctypes.byref(cfg), self.device.index or 0, ctypes.byref(h)))
        self.ctx = h

    def close(self):
        if getattr(self, "ctx", None):
            lib().lk_attn_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        return check(rc, self.ctx, "lk_attn_last_error")

    def device_error(self, stream=None):
        """Synchronise and raise on a recorded device error (a bad page, position, length or tree)."""
        return self._check(lib().lk_attn_get_error(self.ctx, _stream(stream)))

    def rope(self, x, pos, table, rot_offset=0, layout="interleaved", grad=False, out=None, stream=None):
        """x [T][H][head_dim] with [rot_offset, rot_offset + table.rot_dim) of each head rotated to pos [T]; grad: the
        transpose (x is the gradient of the rotated heads, the result that of the plain ones).  out=x works in place."""
        _rows(x, "x", self.device, None, 3)
        _need(x.dtype in _DTYPE, "x: fp32, fp16 or bf16")
        T, H, D = x.shape
        _dense(pos, "pos", (torch.int32,), self.device, T)
        _need(layout in _LAYOUT, "layout: interleaved or half")
        if out is None:
            out = torch.empty(T, H, D, dtype=x.dtype, device=self.device)
        _rows(out, "out", self.device, D, 3)
        _need(out.shape == x.shape and out.dtype == x.dtype, "out: x's shape and dtype")
        self._check(lib().lk_attn_rope(self.ctx, _DTYPE[x.dtype], _ptr(x), x.stride(0), x.stride(1), _ptr(out), out.stride(0),
                                       out.stride(1), T, H, D, rot_offset, table.rot_dim, _LAYOUT[layout], int(grad), _ptr(pos),
                                       _ptr(table.table), table.max_pos, _stream(stream)))
        return out

    def append(self, cache, latent, k_rope, starts, pos, table, layout="interleaved", stream=None):
        """Tokens starts[b] .. starts[b+1]-1 of latent [T][512] and k_rope [T][64] (not yet rotated) become the rows after
        sequence b's lens[b]; cache.pos gets pos [T], cache.mass zeros.  lens stays as it is."""
        T = latent.shape[0]
        _rows(latent, "latent", self.device, ATTN_LATENT, 2)
        _rows(k_rope, "k_rope", self.device, ATTN_ROPE, 2)
        _need(k_rope.shape[0] == T and latent.dtype == k_rope.dtype and latent.dtype in _DTYPE, "latent, k_rope: same rows and dtype")
        _dense(starts, "starts", (torch.int32,), self.device, cache.n_seqs + 1)
        _dense(pos, "pos", (torch.int32,), self.device, T)
        _need(layout in _LAYOUT, "layout: interleaved or half")
        _need(table.rot_dim == ATTN_ROPE, "table: rot_dim %d", ATTN_ROPE)
        self._check(lib().lk_attn_append(self.ctx, cache.struct(), _DTYPE[latent.dtype], _ptr(latent), latent.stride(0),
                                         _ptr(k_rope), k_rope.stride(0), T, _ptr(starts), _ptr(pos), _ptr(table.table),
                                         table.max_pos, _LAYOUT[layout], _stream(stream)))

    def _query(self, q, cache, starts, tree):
        _rows(q, "q", self.device, ATTN_ROW, 3)
        _need(q.dtype == cache.rows.dtype, "q: the cache's dtype")
        _dense(starts, "starts", (torch.int32,), self.device, cache.n_seqs + 1)
        if tree is not None:
            _dense(tree, "tree", (torch.int64, torch.uint64), self.device, q.shape[0])
        return q.shape[0], q.shape[1]

    def tree(self, q, cache, starts, tree, scale, out=None, lse=None, stream=None):
        """out [T][H][512], lse [T][H]: the drafted tokens' attention over their sequence's context and over drafted row j
        where bit j of tree [T] (64-bit words) is set.  tree None: a chain (each token sees the drafts up to itself)."""
        T, H = self._query(q, cache, starts, tree)
        if out is None:
            out = torch.empty(T, H, ATTN_LATENT, dtype=q.dtype, device=self.device)
        if lse is None:
            lse = torch.empty(T, H, device=self.device)
        _rows(out, "out", self.device, ATTN_LATENT, 3)
        _need(out.shape[:2] == q.shape[:2] and out.dtype == q.dtype, "out: [T][H][512] of q's dtype")
        _dense(lse, "lse", (torch.float32,), self.device, T, H)
        self._check(lib().lk_attn_tree(self.ctx, cache.struct(), _ptr(q), q.stride(0), q.stride(1), T, H, _ptr(starts), _ptr(tree),
                                       scale, _ptr(out), out.stride(0), out.stride(1), _ptr(lse), _stream(stream)))
        return out, lse

    def mass(self, q, lse, cache, starts, tree, scale, weight=None, decay=1.0, stream=None):
        """cache.mass = decay * cache.mass + the attention weight that tree() gave each row, summed over heads and over the
        tokens with their weight [T] (0 for rejected drafts; None: 1)."""
        T, H = self._query(q, cache, starts, tree)
        _dense(lse, "lse", (torch.float32,), self.device, T, H)
        if weight is not None:
            _dense(weight, "weight", (torch.float32,), self.device, T)
        self._check(lib().lk_attn_mass(self.ctx, cache.struct(), _ptr(q), q.stride(0), q.stride(1), T, H, _ptr(starts), _ptr(tree),
                                       scale, _ptr(lse), _ptr(weight), decay, _stream(stream)))

    def evict(self, cache, budget, next_pos, sinks=0, recent=0, new_lens=None, stream=None):
        """Cut every sequence to its `budget` best rows (position < sinks or >= next_pos - recent first, then the largest
        mass, then row order); kept rows beyond the budget fill the holes before it.  Returns new_lens [n_seqs], which may
        be cache.lens itself."""
        _dense(next_pos, "next_pos", (torch.int32,), self.device, cache.n_seqs)
        if new_lens is None:
            new_lens = torch.empty(cache.n_seqs, dtype=torch.int32, device=self.device)
        _dense(new_lens, "new_lens", (torch.int32,), self.device, cache.n_seqs)
        self._check(lib().lk_attn_evict(self.ctx, cache.struct(), budget, sinks, recent, _ptr(next_pos), _ptr(new_lens), _stream(stream)))
        return new_lens
