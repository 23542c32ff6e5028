"""A paged cache of keys and values over torch tensors (host-side wrapper of tb_kv_append, tb_kv_read, tb_attention_paged).

The pools, the page table and every array of a batch are the caller's: this class checks them once, keeps them alive and
passes their addresses on.  Calls run on torch's current stream of the pools' device, which has to be the current one.
"""
import ctypes as C

import torch

from . import lib

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_device_of, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _need(ok, text, *args):
    if not ok:
        raise lib.TbError(text % args)


def _ld(t, dtype, width, index):
    """Leading dimension of a matrix of `width` columns whose rows are contiguous; 0 for anything else."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not dtype or len(shape) != 2 or shape[1] != width or t.get_device() != index or (stride[1] != 1 and width != 1):
        return 0
    return stride[0] if shape[0] > 1 else width


def _flat(t, dtype, count, index):
    return t.dtype is dtype and t.numel() == count and t.get_device() == index and t.is_contiguous()


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
        self._index = K.get_device()

    def _batch(self, starts, lens):
        _need(_flat(starts, _I32, self.seqs + 1, self._index) and _flat(lens, _I32, self.seqs, self._index),
              "batch arrays have to be contiguous int32 on %s: %d row starts, %d lengths", self.device, self.seqs + 1, self.seqs)

    def _rows(self, name, t, dtype, width):
        ld = _ld(t, dtype, width, self._index)
        if ld == 0:
            raise lib.TbError("%s has to be %s [rows, %d] on %s with contiguous rows" % (name, dtype, width, self.device))
        return ld

    def _stream(self):
        if _device_of() != self._index:
            raise lib.TbError("the cache is on %s, which is not the current device" % self.device)
        return _stream_of(self._index)

    def append(self, qkv, q, q_start, kv_len, cos=None, sin=None, form=lib.ROPE_PAIRS):
        """qkv: [rows, (query heads + 2 heads) * head_dim] float32 or bfloat16; q: [rows, query heads * head_dim] bfloat16 receives the
        rotated queries; cos, sin: float32 [positions, rotated / 2] or None; q_start, kv_len: as in include/turkce_b200.h."""
        dim, kind = self.head_dim, qkv.dtype
        rows, width = q.shape
        q_heads = width // dim
        ld_q = self._rows("q", q, _BF16, q_heads * dim)
        ld = self._rows("qkv", qkv, kind, (q_heads + 2 * self.heads) * dim)
        if (kind is not _F32 and kind is not _BF16) or qkv.shape[0] != rows:
            raise lib.TbError("qkv has to be float32 or bfloat16, with the %d rows of q" % rows)
        positions = half = 0
        c = d = None
        if cos is not None or sin is not None:
            _need(cos is not None and sin is not None and cos.dim() == 2 and cos.shape == sin.shape, "cos and sin have to be alike")
            positions, half = cos.shape
            if not (_flat(cos, _F32, positions * half, self._index) and _flat(sin, _F32, positions * half, self._index)):
                raise lib.TbError("cos and sin have to be contiguous float32 [positions, rotated / 2] on %s" % self.device)
            if half:
                c, d = cos.data_ptr(), sin.data_ptr()
        self._batch(q_start, kv_len)
        rc = self._lib.tb_kv_append(self._ref, q_start.data_ptr(), kv_len.data_ptr(), qkv.data_ptr(), 1 if kind is _BF16 else 0, ld, rows, q_heads,
                                    c, d, positions, 2 * half, form, q.data_ptr(), ld_q, self._stream())
        if rc:
            lib.check(rc)

    def read(self, start, k, v, first=None):
        """Rows start[s] .. of k and v (bfloat16 [rows, heads * head_dim]; either may be None) from keys first[s] (default 0) on."""
        some = k if k is not None else v
        _need(some is not None, "k or v has to be given")
        width = self.heads * self.head_dim
        ld = self._rows("k and v", some, _BF16, width)
        if some is k and v is not None and (self._rows("k and v", v, _BF16, width) != ld or k.shape != v.shape):
            raise lib.TbError("k and v have to be laid out alike")
        if not _flat(start, _I32, self.seqs + 1, self._index):
            raise lib.TbError("row starts have to be contiguous int32 [%d] on %s" % (self.seqs + 1, self.device))
        if first is not None:
            self._batch(start, first)
        rc = self._lib.tb_kv_read(self._ref, start.data_ptr(), lib._ptr(first), some.shape[0], k.data_ptr() if k is not None else None,
                                  v.data_ptr() if v is not None else None, ld, self.head_dim, self._stream())
        if rc:
            lib.check(rc)

    def workspace(self, q_heads, rows, max_q, max_kv):
        """The memory that `attend` needs for any batch of no more rows, new rows and keys (None: none).  One for every call that may run
        beside another; those that follow one another may share it, whatever their sizes."""
        _need(_device_of() == self._index, "the cache is on %s, which is not the current device", self.device)
        lib.init(self._index)
        n = self._lib.tb_attention_paged_workspace(self._ref, rows, q_heads, max_q, max_kv)
        lib.check(-1 if n < 0 else 0)
        return torch.zeros(n, dtype=torch.uint8, device=self.device) if n else None

    def attend(self, q, att, q_start, kv_len, max_q, max_kv, scale=None, lse=None, workspace=None):
        """att = causal attention of q over the cache (both bfloat16 [rows, query heads * head_dim]); lse: optional float32
        [rows, query heads]; max_q, max_kv: the most new rows and keys a sequence has; scale: 1 / sqrt(head_dim) by default."""
        dim = self.head_dim
        rows, width = q.shape
        q_heads = width // dim
        ld_q = self._rows("q", q, _BF16, q_heads * dim)
        ld_att = self._rows("att", att, _BF16, q_heads * dim)
        if att.shape[0] != rows:
            raise lib.TbError("q and att have to be of one shape")
        sums = room = None
        room_bytes = 0
        if lse is not None:
            if not _flat(lse, _F32, rows * q_heads, self._index):
                raise lib.TbError("lse has to be contiguous float32 [%d, %d] on %s" % (rows, q_heads, self.device))
            sums = lse.data_ptr()
        if workspace is not None:
            if workspace.get_device() != self._index or not workspace.is_contiguous():
                raise lib.TbError("the workspace has to be contiguous on %s" % self.device)
            room, room_bytes = workspace.data_ptr(), workspace.nbytes
        self._batch(q_start, kv_len)
        rc = self._lib.tb_attention_paged(self._ref, q_start.data_ptr(), kv_len.data_ptr(), q.data_ptr(), ld_q, rows, q_heads, max_q, max_kv,
                                          dim ** -0.5 if scale is None else scale, att.data_ptr(), ld_att, sums, room, room_bytes, self._stream())
        if rc:
            lib.check(rc)
