"""CPU tests of the spectrogram cache and dropout: the frame's layout, the refusal rules of the C side (host logic) and of the Python
side.  Nothing here touches a device."""
import ctypes
import math

import numpy as np
import pytest

import cache_reference as ref


@pytest.fixture(scope="module")
def L():
    from gomel_amd import _lib
    return _lib.lib()


def cfg(L, K):
    from gomel_amd._lib import GomelConfig
    c = GomelConfig()
    L.gomel_default_config(ctypes.byref(c))
    c.num_mels = K
    return c


def test_frame_bytes(L):
    for K in (1, 7, 80, 81, 160, 192, 193, 1000, 16384):
        c = cfg(L, K)
        for bits in (8, 4):
            for g in (0, 8, 16, 32, 64):
                codes = (2 * K if bits == 8 else K) + 15 & ~15
                groups = 1 if g == 0 else -(-K // g)
                assert L.gomel_cache_frame_bytes(ctypes.byref(c), bits, g) == (codes + 8 * groups + 15 & ~15)
        for bits, g in ((7, 0), (0, 0), (16, 0), (8, 1), (8, 24), (4, 128), (8, -8)):
            assert L.gomel_cache_frame_bytes(ctypes.byref(c), bits, g) == 0
    assert L.gomel_cache_frame_bytes(None, 8, 0) == 0
    for K in (0, -1, 16385):
        assert L.gomel_cache_frame_bytes(ctypes.byref(cfg(L, K)), 8, 0) == 0


def test_null_arguments(L):
    out, n = ctypes.c_void_p(), ctypes.c_uint64()
    assert L.gomel_cache_create(None, 4, 8, 0, ctypes.byref(out)) == 7
    assert L.gomel_cache_destroy(None) == 0
    assert L.gomel_cache_write(None, 1, 16, 4, 1, None, 0, None, 0, None) == 7
    assert L.gomel_cache_read(None, 1, 16, 4, 1, None, 0, 0.0, 0, 0, None) == 7
    assert L.gomel_cache_bad_slots(None, ctypes.byref(n)) == 7
    assert L.gomel_batch_upload_cache(None, None, None, None, None, None) == 7
    assert L.gomel_to_mel_cache(None, 0, None, None, None, None, 0, None) == 7
    assert L.gomel_dropout(None, 1, 16, 1, 16, 1, 1, 1, 0.5, 0, 0, None) == 7
    assert L.gomel_dropout_backward(None, 1, 16, 1, 16, 1, 1, 1, 0.5, 0, 0, None) == 7


def _hidden(L, name, res, args):
    fn = getattr(L, name)
    fn.restype, fn.argtypes = res, args
    return fn


def test_rows_rule(L):
    """Which input / output rows a call may take: checked against the sets of bytes themselves."""
    ok = _hidden(L, "gomel_debug_rows_ok", ctypes.c_int, [ctypes.c_uint64, ctypes.c_size_t, ctypes.c_uint64, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t])
    rng = np.random.default_rng(5)
    seen = set()
    for _ in range(4000):
        rows, cols, esz = int(rng.integers(1, 5)), int(rng.integers(1, 5)), int(rng.choice([2, 4, 8]))
        sa, sb = (cols + int(rng.integers(0, 7)) for _ in range(2))
        if rng.random() < 0.6:
            sb = sa
        a = 1000 * esz
        b = a + int(rng.integers(-30, 31)) * esz
        cells = [{p + (r * s + k) * esz for r in range(rows) for k in range(cols)} for p, s in ((a, sa), (b, sb))]
        got = ok(a, sa, b, sb, rows, cols, esz)
        if a == b and (sa == sb or rows == 1):
            assert got == 1
        elif cells[0] & cells[1]:
            assert got == 0, (rows, cols, esz, sa, sb, b - a)       # never allowed when an element is shared
        elif sa == sb:
            lo, hi = min(a, b), max(a, b)
            wraps = (hi - lo) % (sa * esz)
            if wraps and cols * esz <= wraps <= (sa - cols) * esz:
                assert got == 1
        seen.add(got)
    assert seen == {0, 1}
    assert ok(64, 3, 4096, 3, 1, 4, 4) == -1 and ok(64, 4, 4096, 3, 2, 4, 4) == -1        # rows that overlap themselves
    assert ok(64, 4, 4096, 4, 0, 4, 4) == -1 and ok(64, 1 << 60, 4096, 4, 2, 4, 4) == -1


def test_drop_rule(L):
    f = _hidden(L, "gomel_debug_drop_rule", ctypes.c_int, [ctypes.c_double, ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_double)])
    below, everything, scale = ctypes.c_uint32(), ctypes.c_int32(), ctypes.c_double()
    for p in (0.0, 1e-12, 2.0 ** -33, 2.0 ** -32, 0.1, 0.5, 0.9, 1 - 2.0 ** -32, 1 - 2.0 ** -34, 1.0):
        assert f(p, ctypes.byref(below), ctypes.byref(everything), ctypes.byref(scale)) == 1
        t = int(np.rint(p * 2.0 ** 32))
        assert bool(everything.value) == (t == 2 ** 32)
        if t < 2 ** 32:
            assert below.value == t and scale.value == 1 / (1 - p)
        else:
            assert scale.value == 0
    for p in (-1e-9, 1.0000001, math.nan, math.inf, -math.inf):
        assert f(p, ctypes.byref(below), ctypes.byref(everything), ctypes.byref(scale)) == 0


def test_reference_generator_is_the_initial_signals():
    """The reference's words are splitmix64 of the index, as gomel_from_mel's x0 documents: its top 53 bits make x0."""
    import gomel_oracle
    x0 = gomel_oracle.x0_splitmix(77, 16)
    for i, v in enumerate(x0):
        halves = []
        for h in (0, 1):
            lo, hi = 0, 2 ** 32
            while hi - lo > 1:                    # smallest t with u < t is u + 1
                mid = (lo + hi) // 2
                if ref.dropped(mid / 2.0 ** 32, 77, 2 * i + h, 1)[0]:
                    hi = mid
                else:
                    lo = mid
            halves.append(lo)
        assert ((halves[1] << 32 | halves[0]) >> 11) * 2.0 ** -53 == v


class _Engine:
    class cfg:
        device = 0
        num_mels = 4
    _h = None


def _cache(K=4):
    from gomel_amd import Cache
    c = object.__new__(Cache)
    c._c, c.num_mels, c.device, c.n_slots = ctypes.c_void_p(), K, 0, 8

    def called(*a):
        raise AssertionError("the library was reached")
    c._write = c._read = called
    return c


def test_python_refuses_what_is_not_rows_of_frames():
    from gomel_amd import DevicePointer
    c = _cache()
    ok = np.zeros((3, 4, 2))
    wide = np.zeros((3, 10, 2))
    for bad in (np.zeros((3, 4)), np.zeros((3, 4, 2), np.int32), np.zeros((4, 3, 2)).transpose(1, 0, 2), np.zeros((3, 4, 2))[:, :, ::-1],
                np.zeros((2, 5)), wide[:, ::2, :], np.zeros((3, 4, 2), dtype=">f8"), ok[::-1], DevicePointer(64, 9, "float32"), DevicePointer(64, 8, "int64")):
        with pytest.raises(ValueError):
            c.write(bad)
        with pytest.raises(ValueError):
            c.read(bad)
    with pytest.raises(TypeError):
        c.write([[0.0] * 8])
    for slots in ([1, 2], [0.0, 1.0, 2.0], np.zeros(4, np.int64), DevicePointer(64, 3, "float64"), DevicePointer(64, 2, "int64")):
        with pytest.raises(ValueError):
            c.write(ok, slots=slots)
        with pytest.raises(ValueError):
            c.read(ok, slots=slots)
    with pytest.raises(ValueError):
        c.write(ok, values=np.zeros((3, 4, 2), np.float32))
    with pytest.raises(ValueError):
        c.write(ok, values=np.zeros((2, 4, 2)))
    with pytest.raises(ValueError):
        c.write(ok, first=-1)
    frozen = np.zeros((3, 4, 2))
    frozen.flags.writeable = False
    with pytest.raises(ValueError):
        c.read(frozen)
    with pytest.raises(ValueError):
        c.write(ok, values=frozen)


def test_python_takes_rows_apart():
    from gomel_amd.cache import _rows
    wide = np.zeros((5, 10, 2), np.float32)
    assert _rows(wide[:, 3:7], 8, "x")[1:4] == (1, 20, 5)
    assert _rows(wide[::2, 3:7], 8, "x")[1:4] == (1, 40, 3)
    assert _rows(np.zeros((20, 2)), 8, "x")[1:4] == (0, 8, 5)
    assert _rows(np.zeros((2, 3, 4, 2), np.float16), 8, "x")[1:4] == (2, 8, 6)
    assert _rows(np.zeros((0, 4, 2)), 8, "x")[3] == 0
    assert _rows(np.zeros((1, 4, 2)), 8, "x")[1:4] == (0, 8, 1)
    with pytest.raises(ValueError):
        _rows(np.zeros((4, 6, 4, 2))[:, :3], 8, "x")          # two outer steps that do not join into one
    with pytest.raises(ValueError):
        _rows(np.broadcast_to(np.zeros((1, 4, 2)), (3, 4, 2)), 8, "x")


def test_python_refuses_dropout_of_other_arrays():
    from gomel_amd import cache
    x = np.zeros((3, 4), np.float32)
    for bad in (np.zeros((3, 4), np.int64), x.T, x[:, ::2]):
        with pytest.raises(ValueError):
            cache.dropout(_Engine, bad, 0.5, 1)
    for out in (np.zeros((4, 3), np.float32), np.zeros((3, 4)), np.zeros(12, np.float32)):
        with pytest.raises(ValueError):
            cache.dropout(_Engine, x, 0.5, 1, out=out)
    from gomel_amd import DevicePointer
    with pytest.raises(ValueError):
        cache.dropout(_Engine, DevicePointer(64, 8, "float32"), 0.5, 1)


def test_torch_tensors_on_the_cpu_are_refused():
    torch = pytest.importorskip("torch") if "torch" in __import__("sys").modules else None
    if torch is None:
        class Fake:                                           # the session does not import torch: what such a tensor looks like
            is_cuda, dtype, shape = False, "torch.float32", (3, 4, 2)

            def data_ptr(self):
                return 64
        t = Fake()
    else:
        t = torch.zeros(3, 4, 2)
    with pytest.raises(ValueError):
        _cache().write(t)


def test_reference_quantiser_at_borders():
    """Ties go to the even code, half a step bounds the error, the definition's special groups."""
    x = np.zeros((1, 4, 2))
    x[0, :, 0], x[0, :, 1] = [0, 15, 0.5, 1.5], [2.5, 14.5, np.nextafter(0.5, 1), np.nextafter(1.5, 0)]
    q, lo, step = ref.quantise(x, 4, 0)
    assert lo[0, 0] == 0 and step[0, 0] == 1
    assert q[0, :, 0].tolist() == [0, 15, 0, 2] and q[0, :, 1].tolist() == [2, 14, 1, 1]
    y = np.random.default_rng(0).normal(size=(5, 81, 2))
    for bits in (8, 4):
        for g in (0, 8, 64):
            _, _, st = ref.quantise(y, bits, g)
            assert np.all(np.abs(ref.stands_for(y, bits, g) - y) <= st[:, np.arange(81) // (g or 81), None] * 0.5000001 + 1e-6)
