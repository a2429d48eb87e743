"""Host-side API of the latent-cache attention operators (include/loki_attn.h): rotary positions, the paged latent
cache, attention of drafted token trees over it, the attention weight of each cached row, and eviction by it.

The cache holds the row that the reference's attention keeps (latent 512, rotated key part 64; src/fused_layer.cu:277-308);
torch supplies device memory and streams, every computation runs in libloki_moe.so.  Calls are queued on the current
stream (or `stream`, whose pool then holds what the call returns) and do not synchronise; AttnContext.device_error()
reports what a kernel refused.
"""
import ctypes

import torch

from . import native as N
from .native import ATTN_LATENT, ATTN_ROPE, ATTN_ROW, check, lib

_DTYPE = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}
_LAYOUT = {"interleaved": N.ROPE_INTERLEAVED, "half": N.ROPE_HALF}
_I32, _F32 = torch.int32, torch.float32


def _need(cond, msg, *args):
    if not cond:
        raise ValueError(msg % args if args else msg)


def _dense(t, name, dtype, device, *shape):
    """A contiguous tensor of this dtype and shape on device number `device`; its address."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous()):
        raise ValueError("%s: a contiguous %s tensor of shape %s on cuda:%d" % (name, dtype, shape, device))
    return t.data_ptr()


def _rows(t, name, device, last):
    """A tensor on device number `device` whose last dimension is dense and `last` wide (None: any); the other strides are
    free.  Its address and strides."""
    if not (isinstance(t, torch.Tensor) and t.get_device() == device):
        raise ValueError("%s: a tensor on cuda:%d" % (name, device))
    st = t.stride()
    if (last is not None and t.shape[-1] != last) or (st[-1] != 1 and t.shape[-1] > 1):
        raise ValueError("%s: a dense last dimension%s" % (name, "" if last is None else " of %d" % last))
    return t.data_ptr(), st


def _elsewhere(name, x, device):
    raise ValueError("%s: on cuda:%d, the context on cuda:%d" % (name, x.device, device))


def _on(stream, device):
    """`stream` as the current one: what the call makes comes from its pool (another's memory may be in use until its queue ends)."""
    _need(stream.device.index == device, "stream: one of cuda:%d", device)
    return torch.cuda.stream(stream)


def _queue(stream, device):
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)
    _need(stream.device.index == device, "stream: one of cuda:%d", device)
    return stream.cuda_stream


class RopeTable:
    """cos and sin of positions 0 .. max_pos-1 ([max_pos][rot_dim / 2][2] fp32), angles in 64 bits.  factor > 1 stretches
    the context: frequencies of fewer than beta_slow turns over orig_ctx are divided by factor, those of more than
    beta_fast are kept, with a linear mix between; cos and sin are multiplied by mscale."""

    def __init__(self, max_pos, rot_dim=ATTN_ROPE, base=10000.0, factor=1.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0,
                 mscale=1.0, device="cuda", stream=None):
        device = torch.device(device)
        self.device = torch.cuda.current_device() if device.index is None else device.index
        self.max_pos, self.rot_dim = max_pos, rot_dim
        cfg = N.LkRopeConfig(rot_dim, base, factor, orig_ctx, beta_fast, beta_slow, mscale)
        with torch.cuda.device(self.device), torch.cuda.stream(None) if stream is None else _on(stream, self.device):
            self.table = torch.empty(max(max_pos, 0), max(rot_dim, 0) // 2, 2, device="cuda:%d" % self.device)
            check(lib().lk_attn_rope_table(None, ctypes.byref(cfg), max_pos, self.table.data_ptr(), _queue(None, self.device)))
        self.address = self.table.data_ptr()


class KvCache:
    """The paged latent cache of n_seqs sequences over caller-owned tensors.

    rows [n_pages * page_size][576] fp16 or bf16 (a row stride above 576 is fine); block_table [n_seqs][pages] int32;
    lens [n_seqs] int32, rows of context; mass fp32 and pos int32 [n_pages * page_size], optional (eviction needs both)."""

    def __init__(self, rows, page_size, block_table, lens, mass=None, pos=None):
        _need(isinstance(rows, torch.Tensor) and rows.is_cuda and rows.dim() == 2, "rows: a 2-d CUDA tensor")
        dev, n = rows.get_device(), rows.shape[0]
        _need(rows.dtype in (torch.float16, torch.bfloat16), "rows: fp16 or bf16")
        at, st = _rows(rows, "rows", dev, ATTN_ROW)
        _need(page_size >= 1 and n % page_size == 0, "rows: %d is not a multiple of the page size %d", n, page_size)
        _need(isinstance(block_table, torch.Tensor) and block_table.dim() == 2, "block_table: [n_seqs][pages]")
        seqs, pages = block_table.shape
        table = _dense(block_table, "block_table", _I32, dev, seqs, pages)
        lens_at = _dense(lens, "lens", _I32, dev, seqs)
        mass_at = None if mass is None else _dense(mass, "mass", _F32, dev, n)
        pos_at = None if pos is None else _dense(pos, "pos", _I32, dev, n)
        self.rows, self.page_size, self.block_table, self.lens, self.mass, self.pos = rows, page_size, block_table, lens, mass, pos
        self.device, self.n_seqs, self.dtype = dev, seqs, rows.dtype
        self._struct = N.LkKvCache(at, st[0], _DTYPE[rows.dtype], page_size, n // page_size, table, pages, seqs, lens_at, mass_at, pos_at)
        self._ref = ctypes.byref(self._struct)

    def struct(self):
        return self._ref


class AttnContext:
    """Workspaces of the attention operators for up to max_seqs sequences and max_tokens drafted tokens per call, on one
    device.  Calls on one context run on one stream at a time."""

    def __init__(self, device=0, max_seqs=64, max_tokens=512):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self.device = device.index or 0
        cfg = N.LkAttnConfig(max_seqs, max_tokens)
        h = ctypes.c_void_p()
        self._lib = lib()
        check(self._lib.lk_attn_create(ctypes.byref(cfg), self.device, ctypes.byref(h)))
        self.ctx = h

    def close(self):
        if getattr(self, "ctx", None):
            self._lib.lk_attn_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        return check(rc, self.ctx, "lk_attn_last_error") if rc else rc

    def device_error(self, stream=None):
        """Synchronise and raise on a recorded device error (a bad page, position, length or tree)."""
        return self._check(self._lib.lk_attn_get_error(self.ctx, _queue(stream, self.device)))

    def rope(self, x, pos, table, rot_offset=0, layout="interleaved", grad=False, out=None, stream=None):
        """x [T][H][head_dim] with [rot_offset, rot_offset + table.rot_dim) of each head rotated to pos [T]; grad: the
        transpose (x is the gradient of the rotated heads, the result that of the plain ones).  out=x works in place."""
        dev = self.device
        if stream is not None:
            with _on(stream, dev):
                return self.rope(x, pos, table, rot_offset, layout, grad, out)
        if table.device != dev:
            _elsewhere("table", table, dev)
        at, st = _rows(x, "x", dev, None)
        _need(x.dim() == 3 and x.dtype in _DTYPE, "x: [T][H][head_dim], fp32, fp16 or bf16")
        _need(layout in _LAYOUT, "layout: interleaved or half")
        T, H, D = x.shape
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
            to, so = out.data_ptr(), (H * D, D)
        else:
            to, so = _rows(out, "out", dev, D)
            _need(out.shape == x.shape and out.dtype is x.dtype, "out: x's shape and dtype")
        rc = self._lib.lk_attn_rope(self.ctx, _DTYPE[x.dtype], at, st[0], st[1], to, so[0], so[1], T, H, D, rot_offset, table.rot_dim,
                                    _LAYOUT[layout], grad, _dense(pos, "pos", _I32, dev, T), table.address, table.max_pos,
                                    _queue(None, dev))
        if rc:
            self._check(rc)
        return out

    def append(self, cache, latent, k_rope, starts, pos, table, layout="interleaved", stream=None):
        """Tokens starts[b] .. starts[b+1]-1 of latent [T][512] and k_rope [T][64] (not yet rotated) become the rows after
        sequence b's lens[b]; cache.pos gets pos [T], cache.mass zeros.  lens stays as it is."""
        dev = self.device
        if cache.device != dev:
            _elsewhere("cache", cache, dev)
        if table.device != dev:
            _elsewhere("table", table, dev)
        at, st = _rows(latent, "latent", dev, ATTN_LATENT)
        kt, ks = _rows(k_rope, "k_rope", dev, ATTN_ROPE)
        _need(latent.dim() == 2 and k_rope.dim() == 2 and k_rope.shape[0] == latent.shape[0] and latent.dtype is k_rope.dtype and
              latent.dtype in _DTYPE, "latent, k_rope: [T] rows of the same dtype")
        _need(layout in _LAYOUT, "layout: interleaved or half")
        _need(table.rot_dim == ATTN_ROPE, "table: rot_dim %d", ATTN_ROPE)
        T = latent.shape[0]
        self._check(self._lib.lk_attn_append(self.ctx, cache._ref, _DTYPE[latent.dtype], at, st[0], kt, ks[0], T,
                                             _dense(starts, "starts", _I32, dev, cache.n_seqs + 1), _dense(pos, "pos", _I32, dev, T),
                                             table.address, table.max_pos, _LAYOUT[layout], _queue(stream, dev)))

    def _query(self, q, cache, starts, tree):
        if cache.device != self.device:
            _elsewhere("cache", cache, self.device)
        at, st = _rows(q, "q", self.device, ATTN_ROW)
        _need(q.dim() == 3 and q.dtype is cache.dtype, "q: [T][H][576] of the cache's dtype")
        tree_at = None
        if tree is not None:
            tree_at = _dense(tree, "tree", torch.uint64 if tree.dtype is torch.uint64 else torch.int64, self.device, q.shape[0])
        return at, st, _dense(starts, "starts", _I32, self.device, cache.n_seqs + 1), tree_at

    def tree(self, q, cache, starts, tree, scale, out=None, lse=None, stream=None):
        """out [T][H][512], lse [T][H]: the drafted tokens' attention over their sequence's context and over drafted row j
        where bit j of tree [T] (64-bit words) is set.  tree None: a chain (each token sees the drafts up to itself)."""
        if stream is not None:
            with _on(stream, self.device):
                return self.tree(q, cache, starts, tree, scale, out, lse)
        at, st, starts_at, tree_at = self._query(q, cache, starts, tree)
        T, H, _ = q.shape
        if out is None:
            out = q.new_empty((T, H, ATTN_LATENT))
            to, so = out.data_ptr(), (H * ATTN_LATENT, ATTN_LATENT)
        else:
            to, so = _rows(out, "out", self.device, ATTN_LATENT)
            _need(out.dim() == 3 and out.shape[:2] == q.shape[:2] and out.dtype is q.dtype, "out: [T][H][512] of q's dtype")
        if lse is None:
            lse = q.new_empty((T, H), dtype=_F32)
            lse_at = lse.data_ptr()
        else:
            lse_at = _dense(lse, "lse", _F32, self.device, T, H)
        rc = self._lib.lk_attn_tree(self.ctx, cache._ref, at, st[0], st[1], T, H, starts_at, tree_at, scale, to, so[0], so[1],
                                    lse_at, _queue(None, self.device))
        if rc:
            self._check(rc)
        return out, lse

    def mass(self, q, lse, cache, starts, tree, scale, weight=None, decay=1.0, stream=None):
        """cache.mass = decay * cache.mass + the attention weight that tree() gave each row, summed over heads and over the
        tokens with their weight [T] (0 for rejected drafts; None: 1).  Sequences without tokens keep theirs.  An expanded q
        (a stride of 0), which tree() takes, is refused here."""
        at, st, starts_at, tree_at = self._query(q, cache, starts, tree)
        T, H, _ = q.shape
        self._check(self._lib.lk_attn_mass(self.ctx, cache._ref, at, st[0], st[1], T, H, starts_at, tree_at, scale,
                                           _dense(lse, "lse", _F32, self.device, T, H),
                                           None if weight is None else _dense(weight, "weight", _F32, self.device, T), decay,
                                           _queue(stream, self.device)))

    def evict(self, cache, budget, next_pos, sinks=0, recent=0, new_lens=None, stream=None):
        """Cut every sequence to its `budget` best rows (position < sinks or >= next_pos - recent first, then the largest
        mass, then row order); kept rows beyond the budget fill the holes before it.  Returns new_lens [n_seqs], which may
        be cache.lens itself."""
        if stream is not None:
            with _on(stream, self.device):
                return self.evict(cache, budget, next_pos, sinks, recent, new_lens)
        if cache.device != self.device:
            _elsewhere("cache", cache, self.device)
        if new_lens is None:
            new_lens = next_pos.new_empty((cache.n_seqs,))
        self._check(self._lib.lk_attn_evict(self.ctx, cache._ref, budget, sinks, recent,
                                            _dense(next_pos, "next_pos", _I32, self.device, cache.n_seqs),
                                            _dense(new_lens, "new_lens", _I32, self.device, cache.n_seqs), _queue(None, self.device)))
        return new_lens
