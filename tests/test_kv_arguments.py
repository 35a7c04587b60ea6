"""What the Python calls of the paged key-value cache refuse before the library is called, which sees addresses only: arrays of another type than the
call reads or writes, arrays that are too short, numbers that 32 bits do not hold."""
from types import SimpleNamespace

import pytest

import tensorwarp_amd as T

KV, DIM, HEADS, SEQS, STRIDE, PAGE, ROWS = 2, 64, 6, 3, 4, 16, 5
WIDTH = HEADS * DIM


def array(dtype, numel):
    return SimpleNamespace(ptr=0x1000, dtype=dtype, numel=numel)


class Device:
    """A device whose library takes every call and keeps its arguments."""

    def __init__(self):
        self.handle, self.calls = 1, []
        take = lambda *args: self.calls.append(args) or 0
        self._l = SimpleNamespace(twm_kv_append=take, twm_attn_decode=take, twm_attn_prompt=take)


@pytest.fixture()
def dev():
    return Device()


def cache(**kw):
    a = dict(k=array("f16", 10 * KV * PAGE * DIM), v=array("f16", 10 * KV * PAGE * DIM), page_tokens=PAGE, kv_heads=KV, head_dim=DIM)
    a.update(kw)
    return T.KvCache(**a)


def seqs(**kw):
    a = dict(tables=array("i32", SEQS * STRIDE), lengths=array("i32", SEQS), seqs=SEQS, table_stride=STRIDE, starts=array("i32", SEQS + 1))
    a.update(kw)
    return T.KvSequences(**a)


def append(dev, **kw):
    a = dict(qkv=array("f32", ROWS * (HEADS + 2 * KV) * DIM), rows=ROWS, q_heads=HEADS, q_out=array("f16", ROWS * WIDTH), cos_sin=array("f32", 100 * DIM),
             positions=100, rotary_dim=DIM)
    a.update(kw)
    return T.kv_append(dev, cache(), seqs(), **a)


def decode(dev, **kw):
    a = dict(q=array("f16", SEQS * WIDTH), q_heads=HEADS, out=array("f16", SEQS * WIDTH))
    a.update(kw)
    return T.attention_decode(dev, cache(), seqs(starts=None), **a)


def prompt(dev, **kw):
    a = dict(q=array("f16", ROWS * WIDTH), rows=ROWS, q_heads=HEADS, out=array("f16", ROWS * WIDTH))
    a.update(kw)
    return T.attention_prompt(dev, cache(), seqs(), **a)


CALLS = [append, decode, prompt]


@pytest.mark.parametrize("call", CALLS)
def test_arrays_that_fit_are_passed_on(dev, call):
    call(dev)
    assert len(dev.calls) == 1


@pytest.mark.parametrize("call,name,wrong", [(append, "q_out", ("f32", "u8", "i32")), (append, "cos_sin", ("f16", "i32")), (decode, "q", ("f32", "u8", "i32")),
                                             (decode, "out", ("f32", "u8", "i32")), (prompt, "q", ("f32", "u8", "i32")), (prompt, "out", ("f32", "u8", "i32"))])
def test_other_types(dev, call, name, wrong):
    for dtype in wrong:
        with pytest.raises(ValueError, match="%s is %s" % (name, dtype)):
            call(dev, **{name: array(dtype, 1 << 20)})
    assert not dev.calls


@pytest.mark.parametrize("call,name,dtype,most", [(append, "qkv", "f32", ROWS * (HEADS + 2 * KV) * DIM), (append, "qkv", "f16", ROWS * (HEADS + 2 * KV) * DIM),
                                                  (append, "q_out", "f16", ROWS * WIDTH), (append, "cos_sin", "f32", 100 * DIM), (decode, "q", "f16", SEQS * WIDTH),
                                                  (decode, "out", "f16", SEQS * WIDTH), (prompt, "q", "f16", ROWS * WIDTH), (prompt, "out", "f16", ROWS * WIDTH)])
def test_short_arrays(dev, call, name, dtype, most):
    with pytest.raises(ValueError, match="%s has %d elements of %d" % (name, most - 1, most)):
        call(dev, **{name: array(dtype, most - 1)})
    assert not dev.calls
    call(dev, **{name: array(dtype, most)})


def test_strides_count(dev):
    for call, rows in ((decode, SEQS), (prompt, ROWS)):
        for name, stride in (("q", "q_stride"), ("out", "out_stride")):
            ends = (rows - 1) * (WIDTH + 8) + WIDTH
            call(dev, **{name: array("f16", ends), stride: WIDTH + 8})
            with pytest.raises(ValueError, match="elements of %d" % ends):
                call(dev, **{name: array("f16", ends - 1), stride: WIDTH + 8})
    ends = (ROWS - 1) * 1000 + (HEADS + 2 * KV) * DIM
    append(dev, qkv=array("f16", ends), qkv_stride=1000)
    with pytest.raises(ValueError, match="elements of %d" % ends):
        append(dev, qkv=array("f16", ends - 1), qkv_stride=1000)
    # no rows, no elements
    prompt(dev, rows=0, q=array("f16", 0), out=array("f16", 0))


def test_descriptions():
    for name, dtype, least in (("tables", "i32", SEQS * STRIDE), ("lengths", "i32", SEQS), ("starts", "i32", SEQS + 1)):
        for wrong in (array("f32", least), array(dtype, least - 1)):
            with pytest.raises(ValueError, match=name):
                seqs(**{name: wrong})
    for name in ("k_scales", "v_scales"):
        for wrong in (array("f16", KV), array("f32", KV - 1)):
            with pytest.raises(ValueError, match=name):
                cache(k=array("u8", 1 << 16), v=array("u8", 1 << 16), **{name: wrong})
    seqs(seqs=0, table_stride=0, tables=array("i32", 0), lengths=array("i32", 0), starts=array("i32", 0))


@pytest.mark.parametrize("wrong", [-1, 1 << 32, (1 << 32) + 5])
def test_numbers_that_32_bits_do_not_hold(dev, wrong):
    # (ctypes would take them modulo 2^32)
    large = array("f16", 1 << 62)
    for call, names in ((append, ("rows", "q_heads", "positions", "rotary_dim", "qkv_stride")), (decode, ("q_heads", "window", "q_stride", "out_stride")),
                        (prompt, ("rows", "q_heads", "window", "q_stride", "out_stride"))):
        for name in names:
            with pytest.raises(ValueError, match=name):
                call(dev, **{name: wrong})
    for name in ("seqs", "table_stride"):
        with pytest.raises(ValueError, match=name):
            seqs(**{name: wrong})
    for name in ("page_tokens", "kv_heads", "head_dim"):
        with pytest.raises(ValueError, match=name):
            cache(k=large, v=large, **{name: wrong})
    assert not dev.calls
