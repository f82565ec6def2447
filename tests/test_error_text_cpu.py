"""mf_last_hip_error from several threads: the calls that hold no state may be made from any number of them on one context, failing ones
among them, and a thread that asks for the text gets a whole one.  No device: mf_shared_expert_static names sizes that it refuses."""
import ctypes as C
import threading
import time

import pytest

from mference_amd import _capi

STATIC_ELEMS = _capi.STATIC_ACT_ELEMS


@pytest.fixture
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def refuse(lib, ctx, f):
    q = _capi.QTensor(1 << 40, 1 << 41, 1 << 42)
    return lib.mf_shared_expert_static(ctx, None, 1 << 43, q, q, q, 4, 64, f, 8, 1 << 44)


def text(f):
    return f"mf_shared_expert_static: t*f = {8 * f} activations exceed the built-in scratch of {STATIC_ELEMS}".encode()


def test_text_of_the_last_error(ctx):
    lib = _capi.lib()
    assert lib.mf_last_hip_error(ctx) == b"" and lib.mf_last_hip_error(None) == b""
    f = STATIC_ELEMS // 8 + 64
    assert refuse(lib, ctx, f) == -4
    assert lib.mf_last_hip_error(ctx) == text(f)
    seen = []
    other = threading.Thread(target=lambda: seen.append(lib.mf_last_hip_error(ctx)))  # the context's text, whichever thread asks
    other.start()
    other.join()
    assert seen == [text(f)]


def test_a_text_stays_until_its_thread_asks_again(ctx):
    lib = C.CDLL(_capi.LIB_PATH)
    lib.mf_last_hip_error.restype, lib.mf_last_hip_error.argtypes = C.c_void_p, [C.c_void_p]
    one, two = STATIC_ELEMS // 8 + 64, 1 << 25
    refuse(_capi.lib(), ctx, one)
    mine = lib.mf_last_hip_error(ctx)
    other = threading.Thread(target=lambda: (refuse(_capi.lib(), ctx, two), lib.mf_last_hip_error(ctx)))
    other.start()
    other.join()
    assert C.string_at(mine) == text(one)
    assert C.string_at(lib.mf_last_hip_error(ctx)) == text(two)


def test_whole_texts_from_several_threads(ctx):
    lib = _capi.lib()
    sizes = (STATIC_ELEMS // 8 + 64, 1 << 25)
    whole, torn, end = {text(f) for f in sizes}, [], time.monotonic() + 2.0
    refuse(lib, ctx, sizes[0])

    def fail(f):
        while time.monotonic() < end:
            refuse(lib, ctx, f)

    def read():
        while time.monotonic() < end and not torn:
            got = lib.mf_last_hip_error(ctx)
            if got not in whole:
                torn.append(got)

    threads = [threading.Thread(target=fail, args=(f,)) for f in sizes] + [threading.Thread(target=read)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not torn, torn
