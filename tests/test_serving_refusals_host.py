"""What the entry points over a paged cache and on logits refuse on the host: every check comes before the device is touched, so
these run without one (the addresses are never followed)."""
import ctypes as C

import pytest

A = 1 << 20             # an address with 16-byte alignment


def struct(**over):
    from turkce_llm_b200 import lib
    c = lib.KvCacheStruct(K=A, V=A, k_scale=None, v_scale=None, table=A, type=0, pages=10, page_size=16, heads=2, head_dim=64, seqs=3, table_ld=5)
    for n, v in over.items():
        setattr(c, n, v)
    return c


def refused(match, name, *args):
    from turkce_llm_b200 import lib
    with pytest.raises(lib.TbError, match=match):
        rc = getattr(lib.load(), name)(*args)
        assert rc != 0
        lib.check(rc)


def append(c, starts=A, lens=A, qkv=A, bf16=0, ld=512, rows=4, heads=4, cos=A, sin=A, positions=9, rot=64, form=0, q=2 * A, ld_q=256):
    return ("tb_kv_append", C.byref(c), starts, lens, qkv, bf16, ld, rows, heads, cos, sin, positions, rot, form, q, ld_q, None)


def attend(c, starts=A, lens=A, q=A, ld_q=256, rows=4, heads=4, max_q=2, max_kv=40, att=2 * A, ld_att=256, lse=None, ws=None, n=0, scale=0.125):
    return ("tb_attention_paged", C.byref(c), starts, lens, q, ld_q, rows, heads, max_q, max_kv, scale, att, ld_att, lse, ws, n, None)


def read(c, starts=A, first=None, rows=4, k=A, v=2 * A, ld_row=128, ld_head=64):
    return ("tb_kv_read", C.byref(c), starts, first, rows, k, v, ld_row, ld_head, None)


@pytest.mark.parametrize("over,match", [
    (dict(K=None), "NULL pool"), (dict(table=None), "NULL pool or table"), (dict(type=2), "unknown cache type"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=136), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=512), "page_size"), (dict(pages=0), "positive"), (dict(heads=-1), "positive"), (dict(seqs=0), "positive"),
    (dict(table_ld=0), "positive"), (dict(pages=1 << 30, heads=4), "2\\^31"), (dict(table_ld=1 << 27), "2\\^31"), (dict(seqs=65536), "65535"),
    (dict(K=A + 8), "aligned"), (dict(type=1), "scale arrays"), (dict(type=1, k_scale=A, v_scale=A + 4), "aligned"),
    (dict(type=1, head_dim=24, k_scale=A, v_scale=A), "multiple of 16"), (dict(k_scale=A), "no scales")])
def test_caches_that_are_none(over, match):
    c = struct(**over)
    for call in (append, attend, read):
        refused(match, *call(c))


@pytest.mark.parametrize("over,match", [
    (dict(starts=None), "batch array"), (dict(lens=None), "batch array"), (dict(qkv=None), "NULL operand"), (dict(q=None), "NULL operand"),
    (dict(rows=-1), "negative"), (dict(heads=3), "cannot share"), (dict(heads=0), "cannot share"), (dict(ld=511), "ld_qkv"), (dict(ld=508), "ld_qkv"),
    (dict(ld=516, bf16=1), "ld_qkv"), (dict(ld_q=255), "ld_q"), (dict(ld_q=260), "ld_q"), (dict(qkv=A + 8), "aligned"), (dict(q=A + 2), "aligned"),
    (dict(rot=63), "rot_dim"), (dict(rot=66), "rot_dim"), (dict(rot=-2), "rot_dim"), (dict(form=2), "rotation form"), (dict(cos=None), "both tables"),
    (dict(sin=None), "both tables"), (dict(positions=0), "both tables"), (dict(q=A), "over the rows")])
def test_append_refuses(over, match):
    refused(match, *append(struct(), **over))


@pytest.mark.parametrize("over,match", [
    (dict(starts=None), "NULL operand"), (dict(lens=None), "NULL operand"), (dict(q=None), "NULL operand"), (dict(att=None), "NULL operand"),
    (dict(rows=-1), "negative"), (dict(max_q=-1), "negative"), (dict(max_kv=-1), "negative"), (dict(heads=5), "cannot share"),
    (dict(ld_q=248), "leading dimensions"), (dict(ld_att=260), "leading dimensions"), (dict(q=A + 8), "aligned"), (dict(ws=A + 4, n=99), "aligned"),
    (dict(att=A), "over the queries"), (dict(heads=260, ld_q=260 * 64, ld_att=260 * 64), "at most 128"), (dict(scale=0.0), "positive and finite"),
    (dict(scale=-1.0), "positive and finite"), (dict(scale=float("inf")), "positive and finite"), (dict(scale=float("nan")), "positive and finite"), (dict(rows=1 << 30), "2\\^31")])
def test_attention_refuses(over, match):
    refused(match, *attend(struct(), **over))


@pytest.mark.parametrize("over,match", [
    (dict(starts=None), "row starts"), (dict(k=None, v=None), "both outputs"), (dict(rows=-1), "negative"), (dict(ld_row=60), "multiples of 8"),
    (dict(ld_head=68), "multiples of 8"), (dict(ld_row=64, ld_head=64), "over one another"), (dict(k=A + 8), "aligned"), (dict(v=A), "over one another")])
def test_read_refuses(over, match):
    refused(match, *read(struct(), **over))


def rules(**over):
    from turkce_llm_b200 import lib
    r = lib.LogitRulesStruct()
    for n, v in over.items():
        setattr(r, n, v)
    return r


@pytest.mark.parametrize("over,call,match", [
    ({}, dict(rows=-1), "rows must be"), ({}, dict(rows=65536), "rows must be"), ({}, dict(vocab=0), "vocab"), ({}, dict(vocab=1 << 30), "vocab"),
    ({}, dict(z=None), "NULL logits"), ({}, dict(out=None), "NULL logits"), ({}, dict(ld=99), "leading dimensions"),
    ({}, dict(ld_out=99), "leading dimensions"), ({}, dict(out=A, ld_out=104), "in place"), ({}, dict(out=A + 64), "overlaps"),
    ({}, dict(out=A - 64), "overlaps"), (dict(prompt=A), {}, "prompt ids need"), (dict(prompt=A, prompt_len=A), {}, "prompt ids need"),
    (dict(output=A, output_len=A, output_ld=1 << 29), {}, "output ids need"), (dict(bias_start=A, bias_entries=3), {}, "bias entries need"),
    (dict(bias_entries=-1), {}, "negative"), (dict(mask=A, masks=4, mask_ld=3), {}, "need 4 words"), (dict(mask=A, masks=3, mask_ld=4), {}, "need mask_row")])
def test_rules_on_logits_refuse(over, call, match):
    a = dict(z=A, ld=100, out=2 * A, ld_out=100, rows=4, vocab=100)
    a.update(call)
    refused(match, "tb_logits_adjust", C.byref(rules(**over)), a["z"], a["ld"], a["out"], a["ld_out"], a["rows"], a["vocab"], None)


def test_null_structs_are_refused():
    refused("NULL cache", "tb_kv_read", None, A, None, 1, A, A, 128, 64, None)
    refused("NULL rules", "tb_logits_adjust", None, A, 100, A, 100, 1, 100, None)


def test_calls_without_rows_do_nothing():
    """(no device is asked for)"""
    from turkce_llm_b200 import lib
    for name, *args in (append(struct(), rows=0, qkv=None, q=None), attend(struct(), rows=0), attend(struct(), max_q=0), read(struct(), rows=0)):
        lib.check(getattr(lib.load(), name)(*args))
    lib.check(lib.load().tb_logits_adjust(C.byref(rules()), None, 100, None, 100, 0, 100, None))


def test_python_wrappers_check_their_tensors():
    import torch
    from turkce_llm_b200 import lib
    from turkce_llm_b200.logit_rules import LogitRules
    from turkce_llm_b200.paged import PagedCache
    K = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(lib.TbError, match="CUDA tensor"):
        PagedCache(K, K, torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(lib.TbError, match="prompt has to be"):
        LogitRules(2, 10, prompt=torch.zeros(2, 3, dtype=torch.int32), prompt_len=torch.zeros(2, dtype=torch.int32))
