"""Which buffers the serving wrappers hand on: truth values do not matter, and
a freed buffer is not one that was left out (no GPU: every call is refused)."""
import pytest

import sheep_amd as sa
from sheep_amd import serving


class At:
    """A made-up device address."""

    def __init__(self, ptr):
        self.ptr = ptr


class Empty(At):
    """A buffer whose truth value says nothing of its memory."""

    def __len__(self):
        return 0


A, B, C, E, FREED = At(1 << 20), At(2 << 20), At(3 << 20), Empty(4 << 20), At(None)
PAGES = dict(k=A, v=B, table=C, n_pages=4, page_size=16, n_seq=2, seq_pages=2, n_kv=2, hd=128)
ADAPTERS = dict(a=A, b=B, n_adapter=2, rank=16, n_in=64, n_out=100)


def test_truth_values_do_not_matter():
    """Each call is refused for what is checked behind its missing buffers."""
    pages, adapters = serving.Pages(**{**PAGES, **dict(k=E, v=E, table=E)}), serving.Adapters(**{**ADAPTERS, **dict(a=E, b=E)})
    with pytest.raises(sa.HipError, match="1024 floats 3 apart"):
        serving.append(pages, E, 1, E, E, E, 8, 4, qkv_stride=3)
    with pytest.raises(sa.HipError, match="512 floats 3 apart"):
        serving.attention(pages, E, E, 8, 4, E, E, q_stride=3)
    with pytest.raises(sa.HipError, match="3 and 0 apart"):
        serving.adjust_logits(E, 2, 100, out=E, tok=E, part=E, stride=3)
    with pytest.raises(sa.HipError, match="without hist_start"):
        serving.adjust_logits(E, 2, 100, out=E, hist=E, n_hist=4, rep=E)
    with pytest.raises(sa.HipError, match="without bias_id"):
        serving.adjust_logits(E, 2, 100, out=E, bias=E, n_bias=4)
    with pytest.raises(sa.HipError, match="1 masks for 2 rows"):
        serving.adjust_logits(E, 2, 100, out=E, mask=E, n_mask=1)
    with pytest.raises(sa.HipError, match="3 and 0 apart"):
        serving.lora(adapters, E, 1, E, E, E, base=E, x_stride=3)


@pytest.mark.parametrize("name", ["seq", "q_out"])
def test_append_refuses_freed_buffers(name):
    with pytest.raises(sa.HipError, match="freed"):
        serving.append(serving.Pages(**PAGES), A, 1, B, C, C, 8, 4, qkv_stride=3, **{name: FREED})


@pytest.mark.parametrize("name", ["out", "tok", "hist", "n_prompt", "rep", "presence", "frequency", "bias_id", "bias",
                                  "bias_start", "mask", "mask_row", "hist_start"])
def test_logits_refuse_freed_buffers(name):
    with pytest.raises(sa.HipError, match="freed"):
        serving.adjust_logits(A, 2, 100, **{**dict(out=B, stride=3), name: FREED})


@pytest.mark.parametrize("name", ["scale", "ranks", "a"])
def test_adapters_refuse_freed_buffers(name):
    with pytest.raises(sa.HipError, match="freed"):
        serving.Adapters(**{**ADAPTERS, name: FREED})


def test_lora_refuses_a_freed_base():
    with pytest.raises(sa.HipError, match="freed"):
        serving.lora(serving.Adapters(**ADAPTERS), A, 1, B, C, C, base=FREED, x_stride=3)


def test_freed_buffers_that_no_call_can_do_without():
    pages = serving.Pages(**PAGES)
    with pytest.raises(sa.HipError, match="missing"):
        serving.append(pages, FREED, 1, B, C, C, 8, 4)
    with pytest.raises(sa.HipError, match="missing"):
        serving.attention(pages, A, B, 8, 4, FREED, C)
    with pytest.raises(sa.HipError, match="missing"):
        serving.adjust_logits(FREED, 2, 100, out=A)
    with pytest.raises(sa.HipError, match="missing"):
        serving.lora(serving.Adapters(**ADAPTERS), A, 1, FREED, C, C)
