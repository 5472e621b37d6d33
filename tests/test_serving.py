"""What the operators of a step of many requests refuse, before any device is
touched, and the sizes of their workspaces (no GPU)."""
import struct

import pytest

import sheep_amd as sa
from sheep_amd import serving


class At:
    """A made-up device address: every call below is refused before it is used."""

    def __init__(self, ptr):
        self.ptr = ptr


A, B, C = At(1 << 20), At(2 << 20), At(3 << 20)
PAGES = dict(k=A, v=B, table=C, n_pages=4, page_size=16, n_seq=2, seq_pages=2, n_kv=2, hd=128)


def refused(match, f, *a, **kw):
    with pytest.raises(sa.HipError, match=match):
        f(*a, **kw)


@pytest.mark.parametrize("change, match", [
    (dict(k=None), "missing pools"), (dict(table=None), "missing pools"), (dict(hd=96), "head_dim 96"),
    (dict(n_kv=0), "0 kv heads"), (dict(page_size=8), "pages of 8"), (dict(page_size=48), "pages of 48"),
    (dict(page_size=131072), "pages of 131072"), (dict(n_pages=0), "0 pages"), (dict(n_seq=0), "0 sequences"),
    (dict(n_seq=65536), "65536 sequences"), (dict(seq_pages=0), "of 0 pages"),
    (dict(seq_pages=1 << 27), "positions a sequence"), (dict(page_stride=4088), "page stride"),
    (dict(page_stride=4100), "page stride"), (dict(k=At(A.ptr + 8)), "16-byte"), (dict(v=At(B.ptr + 2)), "16-byte"),
    (dict(page_size=65536, n_kv=256), "values"),
])
def test_cache_refusals(change, match):
    pg = serving.Pages(**{**PAGES, **change})
    refused(match, serving.append, pg, A, 1, B, C, C, 8, 4)
    refused(match, serving.attention, pg, A, B, 8, 4, C, C)


def test_type_is_checked():
    pg = serving.Pages(**PAGES)
    pg.c = serving._PAGES.pack(A.ptr, B.ptr, C.ptr, 0, 4, 16, 2, 2, 2, 128, 2)
    refused("type 2", serving.append, pg, A, 1, B, C, C, 8, 4)
    ad = serving.Adapters(A, B, 2, 16, 64, 100)
    ad.c = serving._ADAPTERS.pack(A.ptr, B.ptr, 0, 0, 2, 16, 64, 100, -1)
    refused("type -1", serving.lora, ad, A, 1, B, C, C)


@pytest.mark.parametrize("args, kw, match", [
    ((A, -1, B, C, C, 8, 4), {}, "-1 rows"), ((A, (1 << 22) + 1, B, C, C, 8, 4), {}, "4194305 rows"), ((A, 1, B, C, C, 8, 0), {}, "0 heads"),
    ((None, 1, B, C, C, 8, 4), {}, "missing"), ((A, 1, None, C, C, 8, 4), {}, "missing"),
    ((A, 1, B, None, C, 8, 4), {}, "missing"), ((A, 1, B, C, C, 0, 4), {}, "missing"),
    ((A, 1, B, C, C, 8, 4), dict(qkv_stride=1023), "1024 floats 1023 apart"),
])
def test_append_refusals(args, kw, match):
    refused(match, serving.append, serving.Pages(**PAGES), *args, **kw)


@pytest.mark.parametrize("args, kw, match", [
    ((A, B, 8, 3, C, C), {}, "3 heads over 2"), ((A, B, 8, 34, C, C), {}, "34 heads over 2"),
    ((A, B, 8, 0, C, C), {}, "0 heads"), ((A, B, -1, 4, C, C), {}, "lengths up to -1"),
    ((None, B, 8, 4, C, C), {}, "missing"), ((A, None, 8, 4, C, C), {}, "missing"),
    ((A, B, 8, 4, None, C), {}, "missing"), ((A, B, 8, 4, C, None), {}, "missing"),
    ((A, B, 8, 4, C, C), dict(q_stride=511), "511 apart"), ((A, B, 8, 4, At(C.ptr + 8), C), {}, "16-byte"),
])
def test_attention_refusals(args, kw, match):
    refused(match, serving.attention, serving.Pages(**PAGES), *args, **kw)


@pytest.mark.parametrize("kw, match", [
    (dict(n_row=-1), "-1 rows"), (dict(n_row=65536), "65536 rows"), (dict(n_vocab=0), "of 0"),
    (dict(n_vocab=(1 << 30) + 1), "of 1073741825"), (dict(out=None), "missing"), (dict(logits=None), "missing"),
    (dict(tok=B), "missing"), (dict(tok=B, part=At(C.ptr + 8)), "16-byte"), (dict(stride=99), "99 and"),
    (dict(out_stride=99), "99 apart"), (dict(out=A, stride=200), "in place"),
    (dict(hist=C, n_hist=5, rep=C), "hist_start"), (dict(bias=C, n_bias=1, bias_id=C), "bias_start"),
    (dict(bias=C, n_bias=1, bias_start=C), "bias_id"), (dict(mask=C, n_mask=1), "1 masks for 2 rows"),
    (dict(n_hist=-1), "-1 ids"), (dict(n_hist=(1 << 30) + 1), "1073741825 ids"), (dict(n_bias=-2), "-2 biases"),
    (dict(n_mask=-1), "-1 masks"),
])
def test_logits_refusals(kw, match):
    base = dict(logits=A, n_row=2, n_vocab=100, out=B)
    refused(match, serving.adjust_logits, **{**base, **kw})


@pytest.mark.parametrize("change, args, kw, match", [
    (dict(a=None), (), {}, "missing pools"), (dict(rank=12), (), {}, "rank 12"), (dict(rank=264), (), {}, "rank 264"),
    (dict(rank=0), (), {}, "rank 0"), (dict(n_adapter=0), (), {}, "0 of rank"), (dict(n_in=36), (), {}, "36 inputs"),
    (dict(n_out=0), (), {}, "0 outputs"), (dict(a=At(A.ptr + 8)), (), {}, "16-byte"),
    ({}, (A, -1, B, C, C), {}, "-1 rows"), ({}, (A, 65536, B, C, C), {}, "65536 rows"),
    ({}, (None, 1, B, C, C), {}, "missing"), ({}, (A, 1, None, C, C), {}, "missing"),
    ({}, (A, 1, B, None, C), {}, "missing"), ({}, (A, 1, B, C, None), {}, "missing"),
    ({}, (A, 1, B, C, C), dict(x_stride=63), "63 and"), ({}, (A, 1, B, C, C), dict(y_stride=99), "99 apart"),
])
def test_lora_refusals(change, args, kw, match):
    ad = serving.Adapters(**{**dict(a=A, b=B, n_adapter=2, rank=16, n_in=64, n_out=100), **change})
    refused(match, serving.lora, ad, *(args or (A, 1, B, C, C)), **kw)


def test_workspace_sizes():
    assert serving.part_floats(3, 8, 128, 1) == 3 * 8 * 130
    assert serving.part_floats(3, 8, 128, 65) == 3 * 8 * 2 * 130
    assert serving.part_floats(1, 28, 64, 1 << 20) == 28 * 256 * 66
    assert serving.part_floats(0, 8, 128, 1) == serving.part_floats(1, 8, 128, 0) == 0
    assert serving.logits_part_bytes(2, 2049) == 2 * 2 * 16
    assert serving.lora_work_floats(16, 1) == 16 * 32
    assert serving.lora_work_floats(16, 300) == 16 * 8192
    assert serving.lora_work_floats(8, 20000) == 8 * 20000


def test_structures_match_the_header(tmp_path):
    """The packed mirrors have the header's sizes and offsets."""
    import os
    import re
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    mirrors = [
        ("sml_hip_pages", serving._PAGES, "k v table page_stride n_pages page_size n_seq seq_pages n_kv hd type"),
        ("sml_hip_rules", serving._RULES, "hist hist_start n_prompt n_hist rep presence frequency bias_id bias "
         "bias_start n_bias mask mask_row n_mask"),
        ("sml_hip_adapters", serving._ADAPTERS, "a b scale ranks n_adapter rank n_in n_out type")]
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "sml-serve.h"\nint main(void) {\n'
    want = []
    for name, packed, fields in mirrors:
        codes = re.sub(r"(\d+)([a-zA-Z])", lambda m: m[2] * int(m[1]), packed.format)
        assert len(codes) == len(fields.split())
        src += f'printf("%zu\\n", sizeof({name}));\n'
        want.append(packed.size)
        for i, f in enumerate(fields.split()):
            src += f'printf("%zu\\n", offsetof({name}, {f}));\n'
            want.append(struct.calcsize(codes[:i] + "0" + codes[i]))
    (tmp_path / "t.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")],
                   check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True).stdout.split()]
    assert got == want
