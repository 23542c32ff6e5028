"""Penalties, biases and masks on the logits of a batch, over torch tensors (host-side wrapper of tb_logits_adjust).

The arrays are the caller's and may change between calls: this class checks them once, keeps them alive and passes their
addresses on.  Calls run on torch's current stream of the arrays' device, which has to be the current one.
"""
import ctypes as C

import torch

from . import lib
from .paged import _F32, _device_of, _ld, _stream_of


class LogitRules:
    """Rules for `rows` rows of `vocab` logits; every one may be None.

    prompt, output: int32 (or uint32) [rows, ids] with prompt_len, output_len int32 [rows]; repetition, frequency, presence:
    float32 [rows], repetition from 2^-32 to 2^32; bias_start int32 [rows + 1] into bias_id (int32) and bias_value (float32); mask: int32 [masks, words of 32
    tokens], a set bit allows the token, with mask_row int32 [rows] (-1: no mask; None: mask s for row s)."""

    def __init__(self, rows, vocab, prompt=None, prompt_len=None, output=None, output_len=None, repetition=None, frequency=None,
                 presence=None, bias_start=None, bias_id=None, bias_value=None, mask=None, mask_row=None):
        self._lib = lib.load()
        self.rows, self.vocab = rows, vocab
        given = [t for t in (prompt, output, repetition, frequency, presence, bias_id, mask) if t is not None]
        self.device = given[0].device if given else torch.device("cuda", torch.cuda.current_device())
        ints = (torch.int32, torch.uint32)
        entries = bias_id.numel() if bias_id is not None else 0
        for name, t, types, shape in (
                ("prompt", prompt, ints, (rows, None)), ("prompt_len", prompt_len, (torch.int32,), (rows,)),
                ("output", output, ints, (rows, None)), ("output_len", output_len, (torch.int32,), (rows,)),
                ("repetition", repetition, (torch.float32,), (rows,)), ("frequency", frequency, (torch.float32,), (rows,)),
                ("presence", presence, (torch.float32,), (rows,)), ("bias_start", bias_start, (torch.int32,), (rows + 1,)),
                ("bias_id", bias_id, ints, (entries,)), ("bias_value", bias_value, (torch.float32,), (entries,)),
                ("mask", mask, ints, (None, None)), ("mask_row", mask_row, (torch.int32,), (rows,))):
            if t is None:
                continue
            ok = t.is_cuda and t.device == self.device and t.is_contiguous() and t.dtype in types and t.dim() == len(shape) and \
                all(n is None or n == m for n, m in zip(shape, t.shape))
            if not ok:
                raise lib.TbError("%s has to be %s %s, contiguous, on %s" % (name, types[0], shape, self.device))
        for a, b in ((prompt, prompt_len), (output, output_len), (bias_start, bias_id), (bias_id, bias_value)):
            if (a is None) != (b is None):
                raise lib.TbError("ids need their lengths, biases their starts, ids and values")
        if mask_row is not None and mask is None:
            raise lib.TbError("mask_row needs masks")
        if mask is not None and rows and (mask.shape[1] < -(-vocab // 32) or mask.shape[0] < (rows if mask_row is None else 1)):
            raise lib.TbError("masks have to have %d words each, and without mask_row one for each of the %d rows" % (-(-vocab // 32), rows))
        self._kept = (prompt, prompt_len, output, output_len, repetition, frequency, presence, bias_start, bias_id, bias_value, mask, mask_row)
        width = lambda t: t.shape[1] if t is not None else 0  # noqa: E731
        self._struct = lib.LogitRulesStruct(*[lib._ptr(t) if t is not None and t.numel() else None for t in self._kept], width(prompt),
                                            width(output), mask.shape[0] if mask is not None else 0, width(mask), entries)
        self._ref = C.addressof(self._struct)
        self._index = self.device.index

    def apply(self, logits, out=None):
        """out = the rules on logits (float32 [rows, vocab], rows contiguous); out None: in place."""
        out = logits if out is None else out
        rows, vocab = self.rows, self.vocab
        a, b = _ld(logits, _F32, vocab, self._index), _ld(out, _F32, vocab, self._index)
        if a == 0 or b == 0 or logits.shape[0] != rows or out.shape[0] != rows:
            raise lib.TbError("logits have to be float32 [%d, %d] on %s with contiguous rows" % (rows, vocab, self.device))
        if _device_of() != self._index:
            raise lib.TbError("the rules are on %s, which is not the current device" % self.device)
        rc = self._lib.tb_logits_adjust(self._ref, logits.data_ptr(), a, out.data_ptr(), b, rows, vocab, _stream_of(self._index))
        if rc:
            lib.check(rc)
