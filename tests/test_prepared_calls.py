"""Prepared calls of the Python mirror: what the address of a step's rows may be given as (no GPU: the library's function is a
fake that keeps what it gets)."""
import ctypes as C

import pytest


@pytest.fixture
def handle():
    from flint_mac_b200.capi import Attn

    class Fake(Attn):
        def __init__(self):
            self._h, self.got = 1, []

        def close(self):
            self._h = None

        __del__ = close

        def _bound(self, name, *args):
            self.rows = args[3]
            return (lambda *a: self.got.append(self.rows.value) or 0), (), C.create_string_buffer(8)

    return Fake()


@pytest.mark.parametrize("as_what", [int, C.c_void_p, lambda a: C.cast(a, C.POINTER(C.c_float)), lambda a: None])
def test_addresses(handle, as_what):
    call = handle.prepared_decode_dev(0, [0, 1], 0, 4096, 0)
    call(as_what(256))
    call(512)
    assert handle.got == [None if as_what(256) is None else 256, 512]


def test_no_address(handle):
    with pytest.raises((TypeError, C.ArgumentError)):
        handle.prepared_decode_dev(0, [0], 0, 4096, 0)(object())
    assert handle.got == []


def test_closed(handle):
    from flint_mac_b200 import FlintAttnError

    call = handle.prepared_decode_dev(0, [0], 0, 4096, 0)
    handle.close()
    with pytest.raises(FlintAttnError, match="closed"):
        call(256)
