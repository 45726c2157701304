"""The session's configuration and callers compiled against another version of it.  Host only: every call is refused before a device is used."""
import ctypes as C

import pytest

from cavs_amd import session

FIELDS = [f[0] for f in session._Config._fields_]


def _raw():
    """The library by itself, as a C program links it"""
    session.lib()
    l = C.CDLL(session.LIB_PATH)
    l.cavs_session_error.restype = C.c_char_p
    return l


def _bytes(**kw):
    a = dict(model=0, loss=0, opt=2, V=10, E=4, H=8, C=20, device=-5)  # (no such device)
    a.update(kw)
    return bytes(session._Config(**a))


def _create(fn, data, *size):
    h = C.c_void_p()
    buf = C.create_string_buffer(data, len(data))
    l = _raw()
    rc = getattr(l, fn)(buf, *size, C.byref(h))
    assert rc < 0 and not h
    return l.cavs_session_error().decode()


def test_a_program_of_the_smaller_struct_is_not_read_beyond_it():
    """What lies behind the struct of a program compiled before `vocab_head` is the program's own."""
    old = session._Config.vocab_head.offset
    assert FIELDS.index("vocab_head") == FIELDS.index("head_chunks") + 1
    why = _create("cavs_session_create", _bytes()[:old] + b"\xff" * (C.sizeof(session._Config) - old))
    assert "vocab_head" not in why and "optimizer" not in why and "ortho" not in why, why
    # (it got as far as the device)
    assert why == _create("cavs_session_create", _bytes()[:old] + bytes(C.sizeof(session._Config) - old))


@pytest.mark.parametrize("field", ["vocab_head", "optimizer", "ortho_lr"])
def test_a_struct_is_read_as_far_as_its_size(field):
    at, n = getattr(session._Config, field).offset, C.sizeof(session._Config)
    bad = _bytes(**{field: -1})
    assert field in _create("cavs_session_create_sized", bad, C.c_size_t(n)) or field == "optimizer"
    device = _create("cavs_session_create_sized", _bytes(), C.c_size_t(n))
    assert _create("cavs_session_create_sized", bad, C.c_size_t(at)) == device
    assert _create("cavs_session_create_sized", bad, C.c_size_t(n)) != device


def test_sizes_that_are_refused():
    n = C.sizeof(session._Config)
    assert "smaller than any" in _create("cavs_session_create_sized", _bytes(), C.c_size_t(8))
    assert "does not have" in _create("cavs_session_create_sized", _bytes() + b"\0\0\1\0", C.c_size_t(n + 4))
    device = _create("cavs_session_create_sized", _bytes(), C.c_size_t(n))
    assert _create("cavs_session_create_sized", _bytes() + bytes(8), C.c_size_t(n + 8)) == device
