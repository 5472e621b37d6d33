"""A step that serves many requests at once: the ctypes wrappers of
include/sml-serve.h.

Keys and values live in a paged cache (`Pages`): `append` rotates the new
tokens' keys and writes them with their values, `attention` lets one new token
a sequence attend over its pages, `lora` adds each request's adapter beside a
shared projection (`sheep_amd.gemm`), and `adjust_logits` applies penalties,
biases and grammar masks and picks greedily. Buffers are DevBuf or anything
with a device pointer in `.ptr`; workspaces are the caller's, sized by
`part_floats`, `logits_part_bytes` and `lora_work_floats`. `stream` is a
hipStream_t as an int (0: the null stream). The reference has no counterpart:
it keeps one contiguous cache per sequence (sml/sml-run.c:3414-3434) and picks
greedily (sml/sml-run.c:3539-3544).
"""
import ctypes
import struct

from . import HipError, _chk, lib

TYPES = {"f16": 0, "bf16": 1}
_vp, _int, _size, _float = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float


# The header's structures as packed bytes, in the platform's layout: a step
# makes these calls once a layer, and a ctypes.Structure costs a microsecond more.
_PAGES = struct.Struct("PPPN7i0N")            # sml_hip_pages
_RULES = struct.Struct("PPPiPPPPPPiPPi0N")    # sml_hip_rules
_ADAPTERS = struct.Struct("PPPP5i0N")         # sml_hip_adapters


_block = ctypes.c_char_p
_SIGS = [
    ("sml_hip_paged_append", _int, [_block, _vp, _size, _int, _vp, _vp, _vp, _vp, _int, _int, _vp, _vp]),
    ("sml_hip_paged_part_floats", _size, [_int, _int, _int, _int]),
    ("sml_hip_paged_attention", _int, [_block, _vp, _size, _vp, _int, _int, _float, _vp, _vp, _vp]),
    ("sml_hip_logits_part_bytes", _size, [_int, _int]),
    ("sml_hip_logits_adjust", _int, [_vp, _size, _int, _int, _block, _vp, _size, _vp, _vp, _vp]),
    ("sml_hip_lora_work_floats", _size, [_int, _int]),
    ("sml_hip_lora_add", _int, [_block, _vp, _size, _int, _vp, _vp, _vp, _size, _vp, _vp]),
]
class _Calls:
    """The library's functions, bound at their first use."""

    def __getattr__(self, name):
        for n, res, args in _SIGS:
            f = getattr(lib(), n)
            f.restype, f.argtypes = res, args
            setattr(self, n[8:], f)
        return self.__dict__[name]


_call = _Calls()


# A buffer's truth value does not count (it may have a length), and a freed one
# is an error: as NULL it would pass for one that is left out. The buffers that
# no call can do without the library checks itself.

def _at(b):
    """A buffer's device address, 0 for None."""
    return 0 if b is None else b.ptr


def _freed(*buffers):
    """Refuse freed buffers; 0 (those left, of nothing, lie at no address)."""
    if any(b is not None and b.ptr is None for b in buffers):
        raise HipError("a freed buffer")
    return 0


class Pages:
    """One layer's paged cache: pools k and v [n_pages][page_size][n_kv][hd]
    of 16-bit values, table [n_seq][seq_pages] int32. The buffers stay alive
    with the object."""

    def __init__(self, k, v, table, n_pages, page_size, n_seq, seq_pages, n_kv, hd, dtype="f16", page_stride=0):
        self.buffers = (k, v, table)
        self.n_seq, self.n_kv, self.hd = n_seq, n_kv, hd
        try:
            self.c = _PAGES.pack(_at(k), _at(v), _at(table), page_stride, n_pages, page_size, n_seq, seq_pages, n_kv,
                                 hd, TYPES[dtype])
        except struct.error:
            _freed(k, v, table)
            raise


def append(pages, qkv, n_rows, pos, cos, sin, n_rope, n_head, seq=None, q_out=None, qkv_stride=0, stream=0):
    """Rotate n_rows new tokens' q and k by their positions and write their k
    and v to the cache (sml_hip_paged_append); without q_out the rotated q
    goes back to qkv."""
    _chk(_call.paged_append(pages.c, qkv is not None and qkv.ptr, qkv_stride, n_rows,
                            seq is not None and (seq.ptr or _freed(seq)), pos is not None and pos.ptr,
                            cos is not None and cos.ptr, sin is not None and sin.ptr, n_rope, n_head,
                            q_out is not None and (q_out.ptr or _freed(q_out)), stream), "paged append")


def part_floats(n_seq, n_head, hd, max_len):
    """Floats of attention's workspace."""
    return _call.paged_part_floats(n_seq, n_head, hd, max_len)


def attention(pages, q, lens, max_len, n_head, part, out, scale=0.0, q_stride=0, stream=0):
    """out [n_seq][n_head*hd]: one new token a sequence over its first
    lens[b] positions (sml_hip_paged_attention)."""
    _chk(_call.paged_attention(pages.c, q is not None and q.ptr, q_stride, lens is not None and lens.ptr, max_len,
                               n_head, scale, part is not None and part.ptr, out is not None and out.ptr, stream),
         "paged attention")


def logits_part_bytes(n_row, n_vocab):
    """Bytes of adjust_logits' workspace (with tok)."""
    return _call.logits_part_bytes(n_row, n_vocab)


def adjust_logits(logits, n_row, n_vocab, out=None, tok=None, part=None, hist=None, n_hist=0, hist_start=None,
                  n_prompt=None, rep=None, presence=None, frequency=None, bias_id=None, bias=None, n_bias=0,
                  bias_start=None, mask=None, n_mask=0, mask_row=None, stride=0, out_stride=0, stream=0):
    """Penalties, biases and masks on n_row rows of logits into out (which may
    be logits), and each row's greedy pick into tok (sml_hip_logits_adjust)."""
    try:
        r = _RULES.pack(_at(hist), _at(hist_start), _at(n_prompt), n_hist, _at(rep), _at(presence), _at(frequency),
                        _at(bias_id), _at(bias), _at(bias_start), n_bias, _at(mask), _at(mask_row), n_mask)
    except struct.error:
        _freed(hist, hist_start, n_prompt, rep, presence, frequency, bias_id, bias, bias_start, mask, mask_row)
        raise
    _chk(_call.logits_adjust(logits is not None and logits.ptr, stride, n_row, n_vocab, r,
                             out is not None and (out.ptr or _freed(out)), out_stride,
                             tok is not None and (tok.ptr or _freed(tok)), part is not None and part.ptr, stream),
         "logits")


class Adapters:
    """Low-rank adapters of one projection: a [n_adapter][rank][n_in] and
    b [n_adapter][n_out][rank] of one 16-bit type, scale [n_adapter] floats
    and ranks [n_adapter] int32 (None: 1 and rank). The buffers stay alive
    with the object."""

    def __init__(self, a, b, n_adapter, rank, n_in, n_out, dtype="f16", scale=None, ranks=None):
        self.buffers = (a, b, scale, ranks)
        try:
            self.c = _ADAPTERS.pack(_at(a), _at(b), _at(scale), _at(ranks), n_adapter, rank, n_in, n_out, TYPES[dtype])
        except struct.error:
            _freed(a, b, scale, ranks)
            raise


def lora_work_floats(rank, n_row):
    """Floats of lora's workspace."""
    return _call.lora_work_floats(rank, n_row)


def lora(adapters, x, n_row, adapter, y, work, base=None, x_stride=0, y_stride=0, stream=0):
    """y[r] = base[r] + scale * B (A x[r]) with row r's adapter, -1 for none
    (sml_hip_lora_add); base may be y."""
    _chk(_call.lora_add(adapters.c, x is not None and x.ptr, x_stride, n_row, adapter is not None and adapter.ptr,
                        base is not None and (base.ptr or _freed(base)), y is not None and y.ptr, y_stride,
                        work is not None and work.ptr, stream), "lora")
