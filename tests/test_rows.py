"""What the operators of several rows a sequence and of a cache's upkeep refuse,
before any device is touched, and the size of their workspace (no GPU)."""
import os
import re
import struct
import subprocess

import pytest

import sheep_amd as sa
from sheep_amd import serving


class At:
    """A made-up device address: every call below is refused before it is used."""

    def __init__(self, ptr):
        self.ptr = ptr


A, B, C, D, FREED = At(1 << 20), At(2 << 20), At(3 << 20), At(4 << 20), At(None)
PAGES = dict(k=A, v=B, table=C, n_pages=4, page_size=16, n_seq=2, seq_pages=2, n_kv=2, hd=128)
AXIS = bytes(64)


def refused(match, f, *a, **kw):
    with pytest.raises(sa.HipError, match=match):
        f(*a, **kw)


@pytest.mark.parametrize("change, match", [(dict(k=None), "missing pools"), (dict(page_size=48), "pages of 48"), (dict(n_seq=0), "0 sequences")])
def test_the_cache_is_checked(change, match):
    pg = serving.Pages(**{**PAGES, **change})
    refused(match, serving.append_axes, pg, A, 1, B, B, AXIS, C, C, 8, 4)
    refused(match, serving.attention_rows, pg, serving.Rows(A, B, 1, 8), A, 4, C, D)
    refused(match, serving.accept, pg, 1, A, A, A, A, A, 4)
    refused(match, serving.fork, pg, A, 1, A, A, B, B)
    refused(match, serving.compact, pg, 1, A, A)


@pytest.mark.parametrize("args, kw, match", [
    ((A, -1, B, B, AXIS, C, C, 8, 4), {}, "-1 rows"), ((A, 1, B, B, AXIS, C, C, 8, 0), {}, "0 heads"),
    ((None, 1, B, B, AXIS, C, C, 8, 4), {}, "missing"), ((A, 1, None, B, AXIS, C, C, 8, 4), {}, "missing"),
    ((A, 1, B, None, AXIS, C, C, 8, 4), {}, "missing"), ((A, 1, B, B, None, C, C, 8, 4), {}, "missing"),
    ((A, 1, B, B, AXIS, None, C, 8, 4), {}, "missing"), ((A, 1, B, B, AXIS, C, C, 0, 4), {}, "missing"),
    ((A, 1, B, B, AXIS, C, C, 8, 4), dict(n_axis=0), "0 axes"), ((A, 1, B, B, AXIS, C, C, 8, 4), dict(n_axis=5), "5 axes"),
    ((A, 1, B, B, bytes(32), C, C, 8, 4), {}, "axes of 32 pairs"), ((A, 1, B, B, AXIS, C, C, 8, 4), dict(qkv_stride=3), "3 apart"),
    ((A, 1, B, B, AXIS, C, C, 8, 4), dict(seq=FREED), "freed"), ((A, 1, B, B, AXIS, C, C, 8, 4), dict(q_out=FREED), "freed"),
])
def test_append_axes_refusals(args, kw, match):
    refused(match, serving.append_axes, serving.Pages(**PAGES), *args, **kw)


@pytest.mark.parametrize("rows, args, kw, match", [
    (dict(start=None), {}, {}, "missing starts"), (dict(lens=None), {}, {}, "missing starts"), (dict(n_row=-1), {}, {}, "-1 rows"),
    (dict(n_row=65536), {}, {}, "65536 rows"), (dict(max_len=-1), {}, {}, "up to -1"), (dict(tree=A), {}, {}, "0 words"),
    (dict(tree=A, tree_words=2049), {}, {}, "2049 words"), (dict(cap=-1.0), {}, {}, "capped at -1"),
    (dict(cap=1e-44), {}, {}, "capped"), (dict(cap=1e37), {}, {}, "capped"),
    (dict(cap=3e38), {}, dict(scale=1e20), "capped"), (dict(cap=float("nan")), {}, {}, "capped"), (dict(cap=float("inf")), {}, {}, "capped"),
    ({}, dict(n_head=3), {}, "3 heads over 2"), ({}, dict(n_head=34), {}, "34 heads"), ({}, dict(q=None), {}, "missing rows"),
    ({}, dict(part=None), {}, "missing rows"), ({}, dict(out=None), {}, "missing rows"),
    ({}, dict(part=At(C.ptr + 8)), {}, "16-byte"), ({}, {}, dict(q_stride=511), "511 apart"),
])
def test_attention_rows_refusals(rows, args, kw, match):
    r = serving.Rows(**{**dict(start=A, lens=B, n_row=2, max_len=8), **rows})
    refused(match, serving.attention_rows, serving.Pages(**PAGES), r, **{**dict(q=A, n_head=4, part=C, out=D), **args}, **kw)


@pytest.mark.parametrize("name", ["first", "last", "tree", "pos", "slope", "start", "lens"])
def test_rows_refuse_freed_buffers(name):
    with pytest.raises(sa.HipError, match="freed"):
        serving.Rows(**{**dict(start=A, lens=B, n_row=2, max_len=8), name: FREED})


LAYERS = [(dict(n_layer=16385, layer_stride=1 << 20), "16385 layers"), (dict(n_layer=2, layer_stride=4088), "4088 apart"),
          (dict(n_layer=2, layer_stride=4100), "4100 apart"), (dict(n_layer=-1), "-1 layers")]


@pytest.mark.parametrize("kw, match", LAYERS)
def test_layers_are_checked(kw, match):
    pg = serving.Pages(**PAGES)
    refused(match, serving.accept, pg, 1, A, B, A, A, A, 4, **kw)
    refused(match, serving.fork, pg, A, 1, A, A, B, B, **kw)
    refused(match, serving.compact, pg, 1, A, A, **kw)


@pytest.mark.parametrize("change, match", [
    (dict(n_row=-1), "-1 rows"), (dict(n_row=(1 << 22) + 1), "4194305 rows"), (dict(max_kept=0), "0 kept"),
    (dict(max_kept=1025), "1025 kept"), (dict(start=None), "missing"), (dict(lens=None), "missing"), (dict(tok=None), "missing"),
    (dict(parent=None), "missing"), (dict(pick=None), "missing"), (dict(len_out=B), "in place"), (dict(kept=FREED), "freed"),
    (dict(n_kept=FREED), "freed"), (dict(next=FREED), "freed"), (dict(len_out=FREED), "freed"),
])
def test_accept_refusals(change, match):
    refused(match, serving.accept, serving.Pages(**PAGES), **{**dict(n_row=3, start=A, lens=B, tok=C, parent=C, pick=D, max_kept=4), **change})


@pytest.mark.parametrize("change, match", [
    (dict(n_fork=-1), "-1 sequences"), (dict(n_fork=65536), "65536 sequences"), (dict(lens=None), "missing"),
    (dict(parent=None), "missing"), (dict(fresh=None), "missing"), (dict(table_out=None), "missing"), (dict(len_out=None), "missing"),
    (dict(table_out=C), "in place"), (dict(len_out=A), "in place"), (dict(fresh=FREED), "missing"),
])
def test_fork_refusals(change, match):
    refused(match, serving.fork, serving.Pages(**PAGES), **{**dict(lens=A, n_fork=2, parent=B, fresh=B, table_out=D, len_out=D), **change})


@pytest.mark.parametrize("change, match", [
    (dict(n_move=-1), "-1 pages"), (dict(n_move=65535), "65535 pages"), (dict(src=None), "missing"), (dict(dst=None), "missing"),
    (dict(table=FREED), "freed"), (dict(src=FREED), "missing"),
])
def test_compact_refusals(change, match):
    refused(match, serving.compact, serving.Pages(**PAGES), **{**dict(n_move=2, src=A, dst=B), **change})


def test_no_layers_to_fork_or_compact():
    pg = serving.Pages(**PAGES)
    refused("0 layers", serving.fork, pg, A, 1, A, A, B, B, n_layer=0)
    refused("0 layers", serving.compact, pg, 1, A, A, n_layer=0)


def test_sections():
    assert serving.sections(2, 0, 3) == bytes([0, 0, 2, 2, 2])


def test_workspace_size():
    assert serving.rows_floats(1, 8, 8, 32, 128, 4095) == 8 * (2 * 64 + 1) * 32 * 130
    assert serving.rows_floats(16, 416, 8, 32, 128, 8192) == 8 * (2 * 64 + 16) * 128 * 130
    assert serving.rows_floats(9, 3, 3, 3, 64, 1) == 3 * (2 * 171 + 3) * 3 * 66
    assert serving.rows_floats(0, 8, 8, 32, 128, 4095) == serving.rows_floats(1, 0, 8, 32, 128, 4095) == 0


def test_structure_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = "start len first last tree pos slope cap tree_words n_row max_len".split()
    codes = re.sub(r"(\d+)([a-zA-Z])", lambda m: m[2] * int(m[1]), serving._ROWS.format)
    assert len(codes) == len(fields)
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "sml-serve.h"\nint main(void) {\nprintf("%zu\\n", sizeof(sml_hip_rows));\n'
    src += "".join(f'printf("%zu\\n", offsetof(sml_hip_rows, {f}));\n' for f in fields)
    (tmp_path / "t.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True).stdout.split()]
    assert got == [serving._ROWS.size] + [struct.calcsize(codes[:i] + "0" + codes[i]) for i in range(len(fields))]
