"""Refusals of the attention entry points (no GPU: every check comes before the first CUDA call)."""
import ctypes as C

import numpy as np
import pytest

import sptmm_b200 as sp

A = 1 << 20                      # a 16-byte aligned address that is never followed
INV = np.ones(64)


def cache(**kw):
    a = dict(k=A, v=A, n_pages=4, page_size=16, kv_heads=2, head_dim=128, dtype=sp.F16)
    a.update(kw)
    return sp.KVCache(**a)


def rotate(**kw):
    a = dict(QKV=A, T=3, heads=4, kv_heads=2, head_dim=128, positions=A, inv_freq=INV, Q=A, K=A, V=A)
    a.update(kw)
    sp.rotate_heads(**a)


def prompt(**kw):
    a = dict(Q=A, K=A, V=A, out=A, q_offsets=A, k_offsets=A, n_seqs=1, T=4, Tk=4, heads=4, kv_heads=2, head_dim=128)
    a.update(kw)
    sp.attention_prompt(**a)


def decode(**kw):
    a = dict(Q=A, out=A, B=2, heads=4, cache=cache(), lengths=A, table=A, max_pages=2, workspace=A, workspace_bytes=1 << 40)
    a.update(kw)
    sp.attention_decode(**a)


def refused(call, code, text, **kw):
    with pytest.raises(sp.SptmmError) as e:
        call(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


INVALID, UNSUPPORTED = -1, -3


@pytest.mark.parametrize("call", [rotate, prompt])
@pytest.mark.parametrize("code,text,kw", [
    (INVALID, "neither fp16 nor bf16", dict(dtype=sp.F32)),
    (INVALID, "neither fp16 nor bf16", dict(dtype=sp.I8)),
    (INVALID, "query heads", dict(heads=0)),
    (INVALID, "query heads", dict(kv_heads=0)),
    (INVALID, "query heads", dict(heads=5)),
    (INVALID, "query heads", dict(heads=65536, kv_heads=1024)),
    (UNSUPPORTED, "per key head", dict(heads=258)),
    (INVALID, "multiple of 8", dict(head_dim=12)),
    (INVALID, "multiple of 8", dict(head_dim=0)),
    (UNSUPPORTED, "head_dim", dict(head_dim=136)),
    (INVALID, "flags", dict(flags=sp.X_COLMAJOR)),
    (INVALID, "ldq", dict(ldq=504)),
    (INVALID, "ldq", dict(ldq=516)),
    (INVALID, "ldk", dict(ldk=8)),
    (INVALID, "ldv", dict(ldv=260)),
    (INVALID, "null pointer", dict(Q=0)),
    (INVALID, "16-byte aligned", dict(Q=A + 2)),
    (INVALID, "16-byte aligned", dict(K=A + 8)),
])
def test_shapes_types_strides(call, code, text, kw):
    refused(call, code, text, **kw)


@pytest.mark.parametrize("code,text,kw", [
    (INVALID, "input dtype", dict(in_dtype=sp.I8)),
    (INVALID, "rot_dim", dict(inv_freq=np.ones(65))),
    (INVALID, "rot_dim", dict(inv_freq=np.ones(3))),
    (INVALID, "eps", dict(eps=-1.0)),
    (INVALID, "eps", dict(eps=float("nan"))),
    (INVALID, "come together", dict(K=None)),
    (INVALID, "neither packed rows nor a cache", dict(K=None, V=None)),
    (INVALID, "comes with slots", dict(cache=cache())),
    (INVALID, "comes with slots", dict(slots=A)),
    (INVALID, "cache holds", dict(cache=cache(kv_heads=4), slots=A)),
    (INVALID, "cache holds", dict(cache=cache(head_dim=64), slots=A)),
    (INVALID, "cache holds", dict(cache=cache(dtype=sp.BF16), slots=A)),
    (INVALID, "ldqkv", dict(ldqkv=1022)),
    (INVALID, "ldqkv", dict(ldqkv=1026, in_dtype=sp.F16)),
    (INVALID, "null pointer", dict(positions=None)),
    (INVALID, "null pointer", dict(QKV=0)),
    (INVALID, "4-byte aligned", dict(positions=A + 2)),
    (INVALID, "4-byte aligned", dict(slots=A + 1, cache=cache())),
    (INVALID, "16-byte aligned", dict(q_norm=A + 4)),
])
def test_rotate_refusals(code, text, kw):
    refused(rotate, code, text, **kw)


@pytest.mark.parametrize("code,text,kw", [
    (INVALID, "null pointer", dict(q_offsets=0)),
    (INVALID, "null pointer", dict(k_offsets=0)),
    (INVALID, "null pointer", dict(V=None)),
    (INVALID, "4-byte aligned", dict(k_offsets=A + 2)),
    (INVALID, "T=", dict(T=1 << 30)),
    (INVALID, "Tk=", dict(Tk=1 << 30)),
    (UNSUPPORTED, "sequences", dict(n_seqs=65537)),
    (INVALID, "scale", dict(scale=-0.5)),
    (INVALID, "scale", dict(scale=float("nan"))),
    (INVALID, "scale", dict(scale=float("inf"))),
    (INVALID, "ldo", dict(ldo=100)),
])
def test_prompt_refusals(code, text, kw):
    refused(prompt, code, text, **kw)


@pytest.mark.parametrize("code,text,kw", [
    (INVALID, "page_size", dict(cache=cache(page_size=48))),
    (INVALID, "page_size", dict(cache=cache(page_size=8))),
    (INVALID, "cache of 0 pages", dict(cache=cache(n_pages=0))),
    (INVALID, "page_stride", dict(cache=cache(page_stride=4088))),
    (INVALID, "page_stride", dict(cache=cache(page_stride=4100))),
    (INVALID, "31 bits", dict(cache=cache(n_pages=1 << 27))),
    (INVALID, "cache address", dict(cache=cache(k=0))),
    (INVALID, "cache address", dict(cache=cache(v=A + 8))),
    (INVALID, "neither fp16 nor bf16", dict(cache=cache(dtype=sp.F32))),
    (UNSUPPORTED, "head_dim", dict(cache=cache(head_dim=256))),
    (INVALID, "query heads", dict(heads=3)),
    (UNSUPPORTED, "B=", dict(B=65537)),
    (INVALID, "max_pages", dict(max_pages=1 << 28)),
    (INVALID, "prefix_len", dict(prefix_len=0x7fffffff, prefix_table=A)),
    (INVALID, "null pointer", dict(table=None)),
    (INVALID, "null pointer", dict(prefix_len=5)),
    (INVALID, "null pointer", dict(lengths=0)),
    (INVALID, "null pointer", dict(out=0)),
    (INVALID, "16-byte aligned", dict(workspace=A + 8)),
    (INVALID, "workspace", dict(workspace=None)),
    (INVALID, "workspace", dict(workspace_bytes=15)),
    (INVALID, "4-byte aligned", dict(table=A + 2)),
    (INVALID, "4-byte aligned", dict(lengths=A + 3)),
    (INVALID, "ldq", dict(ldq=100)),
    (INVALID, "ldo", dict(ldo=514)),
    (INVALID, "flags", dict(flags=64)),
    (INVALID, "scale", dict(scale=-1.0)),
])
def test_decode_refusals(code, text, kw):
    refused(decode, code, text, **kw)


def test_reserved_word_and_null_params_are_refused():
    c = cache()
    c.struct.reserved = 1
    refused(decode, INVALID, "reserved", cache=c)
    for name in ("sptmm_rotate_heads", "sptmm_attention_prompt", "sptmm_attention_decode"):
        assert getattr(sp.lib, name)(None, 0, None) == INVALID


def test_workspace_size():
    one = sp.attention_decode_workspace(1, 20, 5, 128)
    assert one >= 16 and sp.attention_decode_workspace(64, 20, 5, 128, 8192) >= sp.attention_decode_workspace(64, 20, 5, 128) >= one
    with pytest.raises(ValueError):
        sp.attention_decode_workspace(1, 20, 6, 128)
    with pytest.raises(ValueError):
        sp.attention_decode_workspace(1, 20, 5, 130)
    need = sp.attention_decode_workspace(2, 4, 2, 128)
    refused(decode, INVALID, "%d needed" % need, workspace_bytes=need - 1)


def test_nothing_to_do_is_not_an_error():
    rotate(T=0)
    prompt(T=0)
    prompt(n_seqs=0)
    decode(B=0)


def test_struct_sizes_match_the_header(tmp_path):
    """The ctypes structures lay their fields out as a C compiler lays out the header's."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"sptmm_kv_cache": sp._KVCacheStruct, "sptmm_rotate_params": sp._RotateParams, "sptmm_prompt_params": sp._PromptParams,
             "sptmm_decode_params": sp._DecodeParams}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "sptmm.h"', "int main(void){"]
    for name, cls in names.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        for field, _ in cls._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, field, name, field))
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "return 0;}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    got = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in names.items():
        assert int(got[name]) == C.sizeof(cls), name
        for field, _ in cls._fields_:
            assert int(got[name + "." + field]) == getattr(cls, field).offset, (name, field)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(20, 5, 128), (8, 2, 128), (16, 16, 64), (8, 1, 128), (128, 1, 64), (100, 4, 96), (2, 1, 8)])
def test_workspace_suffices_for_smaller_batches_and_prefixes(heads, kv_heads, head_dim):
    """What is asked for the largest batch and the longest prefix is enough for every smaller one: a call refuses
    nothing that its own batch does not need."""
    for prefix in (0, 1, 128, 129, 700, 2048, 8192, 100000):
        sizes = [sp.attention_decode_workspace(B, heads, kv_heads, head_dim, prefix) for B in range(1, 400)]
        assert sizes == sorted(sizes), [i + 1 for i in range(1, len(sizes)) if sizes[i] < sizes[i - 1]]
    for B in (1, 8, 9, 33, 64, 65, 128, 129, 399):
        sizes = [sp.attention_decode_workspace(B, heads, kv_heads, head_dim, p) for p in (0, 1, 127, 128, 129, 300, 1000, 1900, 5000, 8192, 30000, 1000000)]
        assert sizes == sorted(sizes), (B, sizes)


def test_workspace_of_a_larger_batch_is_taken():
    """The number of bytes that a call with fewer sequences asks for, as its refusal of 15 bytes names it, is no more
    than the size for the larger batch."""
    for big, small, prefix in ((96, 64, 8192), (65, 64, 8192), (129, 128, 8192), (9, 8, 8192), (400, 3, 300)):
        size = sp.attention_decode_workspace(big, 20, 5, 128, prefix)
        with pytest.raises(sp.SptmmError) as e:
            decode(B=small, heads=20, cache=cache(kv_heads=5), prefix_len=prefix, prefix_table=A, workspace_bytes=15)
        need = int(e.value.message.split(" bytes, ")[1].split()[0])
        assert need <= size, (big, small, prefix)
