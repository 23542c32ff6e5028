"""A paged cache of keys and values over torch tensors (host-side wrapper of tb_kv_append, tb_kv_read, tb_attention_paged).

The pools, the page table and every array of a batch are the caller's: this class checks them once, keeps them alive and
passes their addresses on.  Calls run on torch's current stream of the pools' device, which has to be the current one.
"""
import ctypes as C

import torch

from . import lib


def _need(ok, text, *args):
    if not ok:
        raise lib.TbError(text % args)


def _rows(t, dtype, width, name, device):
    """A matrix of `width` columns whose rows are contiguous; its leading dimension."""
    _need(t.dtype == dtype and t.dim() == 2 and t.shape[1] == width and (t.stride(1) == 1 or width == 1) and t.device == device,
          "%s has to be %s [rows, %d] on %s with contiguous rows", name, dtype, width, device)
    return t.stride(0) if t.shape[0] > 1 else max(width, t.stride(0))


class PagedCache:
    """K, V: [pages, heads, page_size, head_dim], bf16, or float8_e4m3fn with k_scale, v_scale float32 [pages, heads, page_size];
    table: int32 [sequences, pages per sequence].  Entries of the table may change between calls."""

    def __init__(self, K, V, table, k_scale=None, v_scale=None):
        self._lib = lib.load()
        e4m3 = K.dtype == torch.float8_e4m3fn
        _need(K.is_cuda and K.dim() == 4 and (e4m3 or K.dtype == torch.bfloat16), "K has to be a CUDA tensor [pages, heads, page_size, "
              "head_dim] of bfloat16 or float8_e4m3fn")
        pages, heads, page, dim = K.shape
        for name, t, shape, dtype in (("K", K, K.shape, K.dtype), ("V", V, K.shape, K.dtype),
                                      ("k_scale", k_scale, (pages, heads, page), torch.float32),
                                      ("v_scale", v_scale, (pages, heads, page), torch.float32)):
            if name.endswith("scale") and not e4m3:
                _need(t is None, "%s: a bfloat16 cache has no scales", name)
                continue
            _need(t is not None and tuple(t.shape) == tuple(shape) and t.dtype == dtype and t.is_contiguous() and t.device == K.device,
                  "%s has to be %s %s, contiguous, on %s", name, dtype, tuple(shape), K.device)
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == K.device and table.is_contiguous(),
              "table has to be int32 [sequences, pages per sequence], contiguous, on %s", K.device)
        self.K, self.V, self.k_scale, self.v_scale, self.table = K, V, k_scale, v_scale, table
        self.device, self.heads, self.head_dim, self.seqs = K.device, heads, dim, table.shape[0]
        self._struct = lib.KvCacheStruct(lib._ptr(K), lib._ptr(V), lib._ptr(k_scale), lib._ptr(v_scale), lib._ptr(table),
                                         lib.KV_E4M3 if e4m3 else lib.KV_BF16, pages, page, heads, dim, self.seqs, table.shape[1])
        self._ref = C.addressof(self._struct)

    def _batch(self, starts, lens):
        """Addresses of the batch arrays."""
        for t, n in ((starts, self.seqs + 1), (lens, self.seqs)):
            _need(t.dtype == torch.int32 and t.numel() == n and t.is_contiguous() and t.device == self.device,
                  "batch arrays have to be int32 on %s: %d row starts, %d lengths", self.device, self.seqs + 1, self.seqs)
        return starts.data_ptr(), lens.data_ptr()

    def _stream(self):
        _need(torch.cuda.current_device() == self.device.index, "the cache is on %s, which is not the current device", self.device)
        return lib._stream()

    def append(self, qkv, q, q_start, kv_len, cos=None, sin=None, form=lib.ROPE_PAIRS):
        """qkv: [rows, (query heads + 2 heads) * head_dim] float32 or bfloat16; q: [rows, query heads * head_dim] bfloat16 receives the
        rotated queries; cos, sin: float32 [positions, rotated / 2] or None; q_start, kv_len: as in include/turkce_b200.h."""
        dim = self.head_dim
        q_heads = q.shape[-1] // dim
        ld_q = _rows(q, torch.bfloat16, q_heads * dim, "q", self.device)
        _need(qkv.dtype in (torch.float32, torch.bfloat16), "qkv has to be float32 or bfloat16")
        ld = _rows(qkv, qkv.dtype, (q_heads + 2 * self.heads) * dim, "qkv", self.device)
        _need(qkv.shape[0] == q.shape[0], "qkv has %d rows, q %d", qkv.shape[0], q.shape[0])
        positions = half = 0
        if cos is not None or sin is not None:
            _need(cos is not None and sin is not None and cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and
                  cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous() and cos.device == sin.device == self.device,
                  "cos and sin have to be float32 [positions, rotated / 2], contiguous, on %s", self.device)
            positions, half = cos.shape
        starts, lens = self._batch(q_start, kv_len)
        lib.check(self._lib.tb_kv_append(self._ref, starts, lens, qkv.data_ptr(), 1 if qkv.dtype == torch.bfloat16 else 0, ld, q.shape[0],
                                         q_heads, lib._ptr(cos) if half else None, lib._ptr(sin) if half else None, positions, 2 * half,
                                         form, q.data_ptr(), ld_q, self._stream()))

    def read(self, start, k, v, first=None):
        """Rows start[s] .. of k and v (bfloat16 [rows, heads * head_dim]; either may be None) from keys first[s] (default 0) on."""
        some = k if k is not None else v
        _need(some is not None, "k or v has to be given")
        lds = [_rows(t, torch.bfloat16, self.heads * self.head_dim, "k and v", self.device) for t in (k, v) if t is not None]
        _need(len(set(lds)) == 1 and (k is None or v is None or k.shape == v.shape), "k and v have to be laid out alike")
        starts, _ = self._batch(start, start[:self.seqs])
        if first is not None:
            self._batch(start, first)
        lib.check(self._lib.tb_kv_read(self._ref, starts, lib._ptr(first), some.shape[0], lib._ptr(k), lib._ptr(v), lds[0], self.head_dim,
                                       self._stream()))

    def workspace(self, q_heads, rows, max_q, max_kv):
        """The memory that `attend` needs for batches within these bounds (None: none).  One for every call that may run beside another."""
        lib.init(self.device.index)
        n = self._lib.tb_attention_paged_workspace(self._ref, rows, q_heads, max_q, max_kv)
        lib.check(-1 if n < 0 else 0)
        return torch.zeros(n, dtype=torch.uint8, device=self.device) if n else None

    def attend(self, q, att, q_start, kv_len, max_q, max_kv, scale=None, lse=None, workspace=None):
        """att = causal attention of q over the cache (both bfloat16 [rows, query heads * head_dim]); lse: optional float32
        [rows, query heads]; max_q, max_kv: the most new rows and keys a sequence has; scale: 1 / sqrt(head_dim) by default."""
        dim = self.head_dim
        q_heads = q.shape[-1] // dim
        ld_q = _rows(q, torch.bfloat16, q_heads * dim, "q", self.device)
        ld_att = _rows(att, torch.bfloat16, q_heads * dim, "att", self.device)
        _need(q.shape == att.shape, "q and att have to be of one shape")
        if lse is not None:
            _need(lse.dtype == torch.float32 and tuple(lse.shape) == (q.shape[0], q_heads) and lse.is_contiguous() and lse.device == self.device,
                  "lse has to be float32 [%d, %d], contiguous, on %s", q.shape[0], q_heads, self.device)
        if workspace is not None:
            _need(workspace.device == self.device and workspace.is_contiguous(), "the workspace has to be on %s", self.device)
        starts, lens = self._batch(q_start, kv_len)
        lib.check(self._lib.tb_attention_paged(self._ref, starts, lens, q.data_ptr(), ld_q, q.shape[0], q_heads, max_q, max_kv,
                                               dim ** -0.5 if scale is None else scale, att.data_ptr(), ld_att, lib._ptr(lse),
                                               lib._ptr(workspace), workspace.numel() * workspace.element_size() if workspace is not None else 0,
                                               self._stream()))
