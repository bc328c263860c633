"""GPU tests of the spectrogram cache (gomel_cache_*) and dropout (gomel_dropout*) against their definitions in numpy float64
(cache_reference.py).  numpy arrays go through the staging buffer, DevicePointers straight to the kernels; torch's part (streams, graphs,
autograd) runs in a child process."""
import ctypes
import threading

import numpy as np
import pytest

import cache_reference as ref

pytestmark = [pytest.mark.gpu]

TYPES = ["float64", "float32", "float16", "bfloat16"]


def engine(K, **kw):
    import gomel_amd
    m = gomel_amd.NewMel()
    m.NumMels, m.MelFmax, m.Window, m.Resolut = K, 16000, 1280, 4096
    for k, v in kw.items():
        setattr(m, k, v)
    return m.engine()


class Dev:
    """Device memory from the runtime's own allocator: arrays up, arrays down."""

    def __init__(self, hip):
        self.hip, self.held = hip, []
        hip.hipMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
        hip.hipFree.argtypes = [ctypes.c_void_p]
        hip.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
        hip.hipMemset.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t]

    def empty(self, n, dtype):
        import gomel_amd
        size = {"float64": 8, "float32": 4, "float16": 2, "bfloat16": 2, "int64": 8}[dtype]
        p = ctypes.c_void_p()
        assert self.hip.hipMalloc(ctypes.byref(p), max(1, n) * size) == 0
        self.held.append(p)
        return gomel_amd.DevicePointer(p.value, n, dtype)

    def up(self, a, dtype):
        a = np.ascontiguousarray(a)
        raw = ref.to_bf16(a) if dtype == "bfloat16" else a.astype(dtype)
        d = self.empty(a.size, dtype)
        assert self.hip.hipMemcpy(d.data_ptr(), raw.ctypes.data, raw.nbytes, 1) == 0
        return d

    def down(self, d, shape):
        raw = np.empty(d.numel(), np.uint16 if d.dtype == "bfloat16" else d.dtype)
        assert self.hip.hipMemcpy(raw.ctypes.data, d.data_ptr(), raw.nbytes, 2) == 0
        return (ref.from_bf16(raw) if d.dtype == "bfloat16" else raw).astype(np.float64).reshape(shape)

    def free(self):
        for p in self.held:
            self.hip.hipFree(p)


@pytest.fixture
def dev(hip):
    d = Dev(hip)
    yield d
    d.free()


def held(a, dtype):
    """The float64 values that `a` has once it is in `dtype`."""
    with np.errstate(over="ignore"):
        return (ref.from_bf16(ref.to_bf16(np.asarray(a, np.float32))) if dtype == "bfloat16" else np.asarray(a).astype(dtype)).astype(np.float64)


def frames(n, K, seed):
    rng = np.random.default_rng(seed)
    x = rng.uniform(np.log(1e-5), np.log(50.0), (n, K, 2))
    x[rng.random((n, 1, 1)).repeat(K, 1).repeat(2, 2) < 0.1] = np.log(1e-5)           # silent frames: all values equal
    return x


# K: one band, odd, one unit short / long of the vector widths, the framework's 80 / 160 / 192, more than a wave holds, the block-wide form
@pytest.mark.parametrize("K", [1, 2, 7, 64, 80, 81, 160, 192, 193, 515, 1100, 2600])
@pytest.mark.parametrize("dtype", TYPES)
def test_write_and_read_match_the_definition(dev, dtype, K):
    e = engine(K, Resolut=8192) if K > 700 else engine(K)
    for bits in (8, 4):
        for group in (0, 8, 16, 32, 64):
            for n in (1, 2, 37):
                x = frames(n, K, K * 100 + n)
                xd = held(x, dtype)
                want, (q, lo, step) = ref.stands_for(xd, bits, group), ref.quantise(xd, bits, group)
                of = np.arange(K) // (group or K)
                bound = np.abs(lo)[:, of, None] + q * step[:, of, None].astype(np.float64)    # |lo| + q*step: what the sum can lose to
                c = e.cache(n + 5, bits, group)
                slots = np.random.default_rng(n).permutation(n + 5)[:n].astype(np.int64)
                src, val, out, at = dev.up(x, dtype), dev.empty(x.size, dtype), dev.empty(x.size, dtype), dev.up(slots, "int64")
                c.write(src, slots=at, values=val)
                c.read(out, slots=at)
                got, back = dev.down(out, x.shape), dev.down(val, x.shape)
                assert ref.close(got, (want, bound), dtype, 1), (bits, group, n, np.abs(got - want).max())
                assert np.array_equal(got, back, equal_nan=True), (bits, group, n)
                wide = dev.empty(x.size, "float64")                          # the codes themselves: fp64 tells them apart
                c.read(wide, slots=at)
                assert ref.close(dev.down(wide, x.shape), (want, bound), "float64", 2), (bits, group, n)
                c.close()
    e.close()


@pytest.mark.parametrize("dtype", ["float64", "float32", "float16"])
def test_host_memory_is_the_same(dev, dtype):
    """numpy arrays, also with rows apart, and several staging pieces, against the device path's bits."""
    e = engine(80)
    c = e.cache(9000, 8, 16)
    n = 9000
    x = frames(n, 80, 3).astype(dtype)
    slots = np.random.default_rng(1).permutation(n).astype(np.int64)
    src, out, at = dev.up(x, dtype), dev.empty(x.size, dtype), dev.up(slots, "int64")
    c.write(src, slots=at)
    c.read(out, slots=at)
    want = dev.down(out, x.shape)
    c2 = e.cache(9000, 8, 16)
    values = np.full_like(x, 7)
    assert c2.write(x, slots=slots, values=values) is values
    assert np.array_equal(values.astype(np.float64), want)
    assert np.array_equal(c2.read(np.empty_like(x), slots=slots).astype(np.float64), want)
    wide = np.full((n, 83, 2), 5, dtype)
    wide[:, 2:82] = x
    c3 = e.cache(9000, 8, 16)
    c3.write(wide[:, 2:82], slots=at, values=wide[:, 2:82])                    # in place, rows apart, slots on the device
    assert np.array_equal(wide[:, 2:82].astype(np.float64), want) and np.all(wide[:, :2] == 5) and np.all(wide[:, 82:] == 5)
    assert np.array_equal(c3.read(np.empty((n * 80, 2), dtype), slots=slots).reshape(x.shape).astype(np.float64), want)
    y = c3.read(np.empty_like(x), slots=slots, p=0.25, seed=11, offset=3)      # the counter runs on through the pieces
    drop = ref.dropped(0.25, 11, 3, x.size).reshape(x.shape)
    assert np.array_equal(y == 0, drop | (want == 0))
    e.close()
    for k in (c, c2, c3):                                                      # a cache outlives its engine
        k.close()


def test_first_instead_of_slots(dev):
    import gomel_amd
    e = engine(81)
    c = e.cache(50, 8, 0)
    x = frames(20, 81, 9).astype(np.float32)
    c.write(x, first=30)
    want = ref.stands_for(x.astype(np.float64), 8, 0)
    got = c.read(np.empty((50, 81, 2), np.float32))
    assert np.all(got[:30] == 0)                                               # never written: zeros
    assert ref.close(got[30:], (want, np.abs(want) + 16), "float32", 1)
    src, out = dev.up(x, "float32"), dev.empty(x.size, "float32")
    c.write(src, first=7)
    c.read(out, first=7)
    assert np.array_equal(dev.down(out, x.shape), got[30:].astype(np.float64))
    for first in (31, 50, 51, 2 ** 40):
        with pytest.raises(gomel_amd.GomelError) as err:
            c.write(x, first=first)
        assert err.value.status == 5
        with pytest.raises(gomel_amd.GomelError):
            c.read(out, first=first)
    c.write(np.empty((0, 81, 2)), first=50)                                    # no frames: no work
    c.read(np.empty((0, 81, 2), np.float16), slots=np.empty(0, np.int64))
    c.close()
    e.close()


@pytest.mark.parametrize("dtype", ["float64", "float32", "bfloat16"])
@pytest.mark.parametrize("bits,group", [(8, 0), (4, 0), (8, 8), (4, 16), (4, 64)])
def test_values_that_are_not_finite(dev, dtype, bits, group):
    K, n = 81, 12
    x = frames(n, K, 4)
    x[1, 3, 1] = np.nan
    x[2, 20, 0] = np.inf
    x[3, 21, 1] = -np.inf
    x[4] = -np.inf
    x[5] = np.inf
    x[6] = -np.inf
    x[6, 80, 0] = np.inf
    x[7] = np.nan
    x[8, :40] = -np.inf
    x[9, 80, 1], x[9, 0, 0] = np.nan, np.inf
    x[10] = -np.inf
    x[10, 17, 1] = 2.5
    xd = held(x, dtype)
    want, (q, lo, step) = ref.stands_for(xd, bits, group), ref.quantise(xd, bits, group)
    of = np.arange(K) // (group or K)
    with np.errstate(invalid="ignore"):
        bound = np.nan_to_num(np.abs(lo)[:, of, None] + q * step[:, of, None].astype(np.float64), nan=0, posinf=0)
    e = engine(K)
    c = e.cache(n, bits, group)
    src, val, out = dev.up(x, dtype), dev.empty(x.size, dtype), dev.empty(x.size, dtype)
    c.write(src, values=val)
    c.read(out)
    got = dev.down(out, x.shape)
    assert np.array_equal(got, dev.down(val, x.shape), equal_nan=True)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    assert ref.close(got, (want, bound), dtype, 1)
    c.close()
    e.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_codes_next_to_a_border(dev, bits):
    """Values at and one unit beside the middle between two codes, in fp64 and fp32, whole steps and steps that are not: every code as
    the definition in 64 bits has it."""
    K, levels = 192, 2 ** bits - 1
    e = engine(K)
    c = e.cache(64, bits, 0)
    rng = np.random.default_rng(8)
    for dtype in ("float64", "float32"):
        x = np.zeros((64, K, 2), dtype)
        for r in range(64):
            lo, span = rng.uniform(-11, 3), rng.uniform(1e-3, 15)
            if r < 8:
                lo, span = 0.0, float(levels) * 2.0 ** (r - 4)
            lo32, hi32 = np.float32(lo), np.float32(lo + span)
            step = np.float32((np.float64(hi32) - np.float64(lo32)) / levels)
            k = rng.integers(0, levels, (K, 2))
            v = (np.float64(lo32) + (k + 0.5) * np.float64(step)).astype(dtype)
            side = rng.integers(-1, 2, (K, 2))
            v = np.where(side < 0, np.nextafter(v, np.array(-np.inf, dtype)), np.where(side > 0, np.nextafter(v, np.array(np.inf, dtype)), v))
            v[0], v[1] = lo32, hi32
            x[r] = v
        want, (q, _, _) = ref.stands_for(x.astype(np.float64), bits, 0), ref.quantise(x.astype(np.float64), bits, 0)
        out = dev.empty(x.size, "float64")
        c.write(dev.up(x, dtype))
        c.read(out)
        assert ref.close(dev.down(out, x.shape), (want, np.abs(want) + 32), "float64", 2), dtype
        assert len(np.unique(q)) == levels + 1
    c.close()
    e.close()


def test_ranges_at_the_ends_of_fp32(dev):
    """Spans of subnormal size, spans of the whole fp32 range, float64 values that fp32 does not hold."""
    K = 16
    big = float(np.finfo(np.float32).max)
    x = np.zeros((7, K, 2))
    rng = np.random.default_rng(3)
    u = rng.random((K, 2))
    u[0] = [0, 1]
    x[0], x[1], x[2] = u * 1e-44, u * 3e-43, -big + u * (2 * big)
    x[2] = np.clip(x[2], -big, big)
    x[3] = (u - 0.5) * 1e300
    x[4] = 1e300
    x[5] = 1e-310 * u
    x[6] = 1.0 + u * 1e-12                                             # equal in fp32, not in fp64
    e = engine(K)
    for bits in (8, 4):
        c = e.cache(7, bits, 0)
        out = dev.empty(x.size, "float64")
        c.write(dev.up(x, "float64"))
        c.read(out)
        want = ref.stands_for(x, bits, 0)
        assert ref.close(dev.down(out, x.shape), (want, np.abs(want) + np.abs(want).max((1, 2), keepdims=True)), "float64", 2)
        c.close()
    e.close()


@pytest.mark.parametrize("n", [2, 3, 130, 2047, 2048, 2049, 5000])
def test_a_slot_named_twice_keeps_the_last_frame(dev, n):
    K = 24
    e = engine(K)
    c = e.cache(700, 8, 8)
    rng = np.random.default_rng(n)
    for trial in range(3):
        x = frames(n, K, trial).astype(np.float32)
        slots = rng.integers(-2, 60 if trial == 1 else 700, n).astype(np.int64)
        if trial == 2:
            slots[:] = 5
        want = c.read(np.empty((700, K, 2), np.float32)).copy()
        good = ref.stands_for(x.astype(np.float64), 8, 8)
        val = dev.up(np.full(x.shape, 3.0), "float32")
        c.write(dev.up(x, "float32"), slots=dev.up(slots, "int64"), values=val)
        got = c.read(np.empty((700, K, 2), np.float32))
        last = {int(s): r for r, s in enumerate(slots) if s >= 0}
        for s, r in last.items():
            want[s] = good[r]
        assert np.allclose(got, want, rtol=2.0 ** -23, atol=2.0 ** -20), (n, trial)
        back = dev.down(val, x.shape)
        assert np.all(back[slots < 0] == 3.0)                                   # padding: the rows of `values` are left alone
        assert np.allclose(back[slots >= 0], good[slots >= 0], rtol=2.0 ** -23, atol=2.0 ** -20)
    c.close()
    e.close()


@pytest.mark.parametrize("K,dtype,group,n", [(515, "float64", 0, 2100), (515, "float64", 32, 4200), (40, "bfloat16", 8, 6000), (1100, "float32", 0, 2048)])
def test_a_slot_named_twice_by_claims(dev, K, dtype, group, n):
    """The same where the frames claim their slots first: the block-wide form, frames cut into segments, many short frames.  Twice, so
    that the claims of one call do not outlive it."""
    e = engine(K, Resolut=8192) if K > 700 else engine(K)
    c = e.cache(900, 8, group)
    rng = np.random.default_rng(n)
    base = frames(16, K, 1)
    good = ref.stands_for(held(base, dtype), 8, group)
    for trial in range(2):
        which = rng.integers(0, 16, n)                       # row r holds frame which[r] of sixteen
        slots = rng.integers(-1, 900, n).astype(np.int64)
        c.write(dev.up(base[which], dtype), slots=dev.up(slots, "int64"))
        got = c.read(np.empty((900, K, 2)))
        last = {int(s): r for r, s in enumerate(slots) if s >= 0}
        for s, r in last.items():
            assert ref.close(got[s], (good[which[r]], np.abs(good[which[r]]) + 32), "float64", 2), (trial, s)
        if trial == 0:
            assert all(np.all(got[s] == 0) for s in range(900) if s not in last)
    c.close()
    e.close()


def test_padding_and_bad_slots(dev):
    import gomel_amd
    K = 80
    e = engine(K)
    c = e.cache(40, 8, 0)
    x = frames(6, K, 1).astype(np.float32)
    c.write(x, first=0)
    for n, slots in ((6, [3, -1, 40, 5, 2 ** 40, -2 ** 62]), (1, [41]), (1, [-1])):
        out = dev.up(np.full((n, K, 2), 9.0), "float32")
        at = dev.up(np.array(slots), "int64")
        c.read(out, slots=at)
        got = dev.down(out, (n, K, 2))
        for r, s in enumerate(slots):
            assert np.all(got[r] == 9.0) if not 0 <= s < 40 else np.any(got[r] != 9.0)
        before = c.read(np.empty((40, K, 2), np.float32))
        assert c.bad_slots() == sum(s >= 40 for s in slots) and c.bad_slots() == 0
        val = dev.up(np.full((n, K, 2), 9.0), "float32")
        c.write(dev.up(x[:n] + 1, "float32"), slots=at, values=val)
        back = dev.down(val, (n, K, 2))
        after = c.read(np.empty((40, K, 2), np.float32))
        for r, s in enumerate(slots):
            assert np.all(back[r] == 9.0) if not 0 <= s < 40 else np.any(back[r] != 9.0)
        same = [s for s in range(40) if s not in slots]
        assert np.array_equal(before[same], after[same])
        assert c.bad_slots() == sum(s >= 40 for s in slots)
        host = np.full((n, K, 2), 9.0, np.float32)
        if any(s >= 40 for s in slots):                                         # in host memory they are refused, and nothing is done
            for call in (lambda: c.read(host, slots=slots), lambda: c.write(x[:n], slots=slots)):
                with pytest.raises(gomel_amd.GomelError) as err:
                    call()
                assert err.value.status == 5
            assert np.all(host == 9.0) and np.array_equal(c.read(np.empty((40, K, 2), np.float32)), after) and c.bad_slots() == 0
    host = np.full((3, K, 2), 9.0)
    c.read(host, slots=[-1, 3, -7])
    assert np.all(host[[0, 2]] == 9.0) and np.any(host[1] != 9.0)
    c.close()
    e.close()


def test_refusals(dev):
    import gomel_amd
    from gomel_amd import _lib
    L = _lib.lib()
    e = engine(16)
    for bits, group in ((7, 0), (8, 12), (4, 128), (8, -1)):
        with pytest.raises(gomel_amd.GomelError) as err:
            e.cache(4, bits, group)
        assert err.value.status == 1
    with pytest.raises(gomel_amd.GomelError) as err:
        e.cache(0)
    assert err.value.status == 4
    with pytest.raises(gomel_amd.GomelError) as err:
        e.cache(2 ** 52)
    assert err.value.status == 1
    c = e.cache(4)
    x = dev.up(np.zeros((4, 16, 2)), "float32")
    W = lambda *a: L.gomel_cache_write(c._c, *a)      # noqa: E731
    p = x.data_ptr()
    assert W(9, p, 32, 4, None, 0, None, 0, None) == 1 and W(-1, p, 32, 4, None, 0, None, 0, None) == 1          # element type
    assert W(1, p, 31, 4, None, 0, None, 0, None) == 3                                                          # rows that overlap
    assert W(1, p, 32, 2 ** 31, None, 0, None, 0, None) == 3                                                    # more rows than a call takes
    assert W(1, None, 32, 4, None, 0, None, 0, None) == 7
    assert W(1, p, 32, 2, None, 0, p + 4, 32, None) == 1 and W(1, p, 32, 2, None, 0, p + 128, 33, None) == 1    # values across frames
    assert W(1, p, 32, 5, None, 0, None, 0, None) == 5
    R = lambda q: L.gomel_cache_read(c._c, 1, p, 32, 4, None, 0, q, 0, 0, None)      # noqa: E731
    for q in (-0.1, 1.1, float("nan")):
        assert R(q) == 1
    D = lambda *a: L.gomel_dropout(e._h, *a)      # noqa: E731
    assert D(1, p, 8, p, 8, 4, 8, 1.5, 0, 0, None) == 1 and D(5, p, 8, p, 8, 4, 8, 0.5, 0, 0, None) == 1
    assert D(1, p, 8, p + 4, 8, 4, 8, 0.5, 0, 0, None) == 1 and D(1, p, 7, p, 8, 4, 8, 0.5, 0, 0, None) == 3
    assert D(1, None, 8, p, 8, 4, 8, 0.5, 0, 0, None) == 7
    assert D(1, None, 8, None, 8, 0, 8, 0.5, 0, 0, None) == 0
    assert W(1, p + 2, 32, 1, None, 0, None, 0, None) == 1 and W(1, p, 32, 1, p + 4, 0, None, 0, None) == 1     # not aligned to their elements
    assert D(1, p + 1, 8, p + 64, 8, 1, 8, 0.5, 0, 0, None) == 1
    host = np.zeros((4, 16, 2), np.float32)
    with pytest.raises(ValueError):
        c.write(host, slots=np.array([0, 1, 2, 2 ** 63], np.uint64))
    c.close()
    e.close()


def test_closed_caches_and_engines_are_refused():
    import gomel_amd
    e = engine(16)
    c = e.cache(4)
    x = np.zeros((1, 16, 2), np.float32)
    b = gomel_amd.Batch(e, [16])
    c.close()
    c.close()
    for call in (lambda: c.write(x), lambda: c.read(x), c.bad_slots, lambda: b.upload_cache(c, [0]), lambda: e.from_cache(c, [[0]])):
        with pytest.raises(gomel_amd.GomelError) as err:
            call()
        assert err.value.status == 7
    b.close()
    e.close()
    for call in (lambda: e.cache(4), lambda: e.dropout(x, 0.5, 1), lambda: e.dropout_backward(x, 0.5, 1)):
        with pytest.raises(gomel_amd.GomelError) as err:
            call()
        assert err.value.status == 7


def test_a_cache_of_more_than_4_gib(dev):
    """Slots whose byte offset does not fit 32 bits."""
    K = 192
    e = engine(K)
    c = e.cache(12_000_000, 8, 0)                                              # 4.8 GB
    assert c.frame_bytes * c.n_slots > 2 ** 32
    slots = np.array([0, 11_999_999, 10_800_000, 2 ** 32 // c.frame_bytes + 1, 1, 2 ** 31 // c.frame_bytes], np.int64)
    x = frames(6, K, 5).astype(np.float32)
    c.write(dev.up(x, "float32"), slots=dev.up(slots, "int64"))
    out = dev.empty(x.size, "float32")
    c.read(out, slots=dev.up(slots[::-1], "int64"))
    want = ref.stands_for(x.astype(np.float64), 8, 0)
    assert ref.close(dev.down(out, x.shape), (want[::-1], np.abs(want[::-1]) + 16), "float32", 1)
    assert np.array_equal(c.read(np.empty((1, K, 2), np.float32), first=11_999_999)[0].astype(np.float64), dev.down(out, x.shape)[4])
    c.close()
    e.close()


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_matches_the_definition(dev, dtype):
    e = engine(80)
    rng = np.random.default_rng(2)
    for n in (1, 2, 7, 8, 9, 255, 4097, 70001):
        x = rng.normal(size=n) * 3
        x[rng.random(n) < 0.05] = np.nan
        x[rng.random(n) < 0.05] = np.inf
        xd = held(x, dtype)
        for p, seed, offset in ((0.0, 1, 0), (0.1, 2 ** 64 - 1, 1), (0.5, 12345, 7), (0.9, 3, 2 ** 64 - 5), (1.0, 4, 0), (2.0 ** -33, 5, 6), (0.25, 6, 2 ** 63)):
            drop = ref.dropped(p, seed, offset, n) if p < 1 else np.ones(n, bool)
            with np.errstate(invalid="ignore", divide="ignore"):
                want = np.where(drop, 0.0, xd / (1 - p) if p < 1 else 0.0)
            for back in (False, True):
                src, out = dev.up(x, dtype), dev.empty(n, dtype)
                (e.dropout_backward if back else e.dropout)(src, p, seed, offset, out=out)
                got = dev.down(out, n)
                assert ref.close(got, want, dtype, 2), (n, p, seed, offset, back)
                assert np.all(got[drop] == 0) and not np.any(np.signbit(got[drop]))
            (e.dropout)(src, p, seed, offset, out=src)                          # in place
            assert np.array_equal(dev.down(src, n), got, equal_nan=True)
        for h in dev.held:
            dev.hip.hipFree(h)
        dev.held = []
    e.close()


def test_dropout_of_rows_apart(dev):
    """Strided rows of every alignment, host arrays, and the counter by dense index whatever the strides."""
    e = engine(80)
    rng = np.random.default_rng(7)
    for cols, stride in ((1, 1), (1, 3), (5, 5), (5, 9), (8, 8), (33, 40), (160, 163), (4099, 4100)):
        for rows in (1, 3, 50):
            for dtype in ("float64", "float32", "float16"):
                wide = rng.normal(size=(rows, stride)).astype(dtype)
                x = wide[:, stride - cols:]
                drop = ref.dropped(0.3, 99, 5, rows * cols).reshape(rows, cols)
                want = np.where(drop, 0.0, x.astype(np.float64) / 0.7)
                got = e.dropout(x, 0.3, 99, 5)
                assert got.shape == x.shape and got.dtype == x.dtype and ref.close(got, want, dtype, 2)
                into = np.full((rows, stride + 2), 4, dtype)
                e.dropout_backward(x, 0.3, 99, 5, out=into[:, :cols])
                assert np.array_equal(into[:, :cols], got) and np.all(into[:, cols:] == 4)
                e.dropout(x, 0.3, 99, 5, out=x)
                assert np.array_equal(x, got)
    a = np.arange(24.0).reshape(2, 3, 4)
    assert np.array_equal(e.dropout(a, 0.5, 1).reshape(-1), e.dropout(a.reshape(-1), 0.5, 1))
    assert e.dropout(np.empty((0, 4)), 0.5, 1).shape == (0, 4) and e.dropout(np.float32([3.0]), 0.0, 1)[0] == 3.0
    e.close()


def test_dropout_gradient(dev):
    """backward against the formula's derivative and against differences of forward (float64: forward is linear in each kept element)."""
    e = engine(80)
    rng = np.random.default_rng(4)
    x, dy = rng.normal(size=301), rng.normal(size=301)
    dx = e.dropout_backward(dy, 0.35, 17, 3)
    drop = ref.dropped(0.35, 17, 3, 301)
    assert np.allclose(dx, np.where(drop, 0, dy / 0.65), rtol=2.0 ** -51, atol=0)
    h = 2.0 ** -10
    for i in range(0, 301, 7):
        up, dn = x.copy(), x.copy()
        up[i] += h
        dn[i] -= h
        d = (np.sum(dy * e.dropout(up, 0.35, 17, 3)) - np.sum(dy * e.dropout(dn, 0.35, 17, 3))) / (2 * h)
        assert abs(d - dx[i]) < 1e-9                # 600 products of size 10, each off by 2^-53: 1e-13 / h
    e.close()


def test_dropout_beyond_32_bit_indexes(dev):
    """A dense array of more than 2^31 elements: the last ones are reached, with their own counters."""
    e = engine(80)
    n = 2 ** 31 + 1003
    d = dev.empty(n, "float16")
    assert dev.hip.hipMemset(d.data_ptr(), 0x3C, n * 2) == 0                    # 0x3C3C = 1.05859375
    e.dropout(d, 0.5, 21, 9, out=d)
    for at in (0, 2 ** 31 - 500, n - 1000):
        raw = np.empty(1000, np.float16)
        assert dev.hip.hipMemcpy(raw.ctypes.data, d.data_ptr() + 2 * at, 2000, 2) == 0
        assert np.array_equal(raw.astype(np.float64), np.where(ref.dropped(0.5, 21, 9 + at, 1000), 0, 2.1171875)), at
    e.close()


def test_more_frames_than_one_launch_takes(dev):
    """200 million one-band frames (the grids go out in parts): dropout, write and read reach the first, the last and those at the seams."""
    e = engine(1)
    n = 200_000_003
    c = e.cache(n, 8, 0)
    x, y = dev.empty(2 * n, "float16"), dev.empty(2 * n, "float16")
    assert dev.hip.hipMemset(x.data_ptr(), 0x3C, 4 * n) == 0                    # 0x3C3C = 1.05859375
    e.dropout(x, 0.5, 33, 0, out=x)
    c.write(x)
    c.read(y)
    seam = (1 << 22) * 32                                                      # blocks of a launch x frames of a block (8 lanes each)
    for at in (0, seam - 500, n - 1000, 2 * (1 << 22) * 8 - 700):
        want = np.where(ref.dropped(0.5, 33, 2 * at, 2000), 0, 2.1171875)
        for d in (x, y):
            raw = np.empty(2000, np.float16)
            assert dev.hip.hipMemcpy(raw.ctypes.data, d.data_ptr() + 4 * at, 4000, 2) == 0
            assert np.allclose(raw.astype(np.float64), want, rtol=2.0 ** -10, atol=0), at   # lo and lo + 255 * step: one fp16 rounding
    c.close()
    e.close()


@pytest.mark.parametrize("K,bits,group", [(80, 8, 0), (81, 4, 16), (192, 8, 64), (515, 4, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_read_with_dropout_is_dropout_of_the_read(dev, dtype, K, bits, group):
    e = engine(K)
    n = 77
    c = e.cache(n, bits, group)
    x = frames(n, K, 2)
    c.write(dev.up(x, dtype))
    slots = np.random.default_rng(0).permutation(n).astype(np.int64)
    slots[5] = -1
    at = dev.up(slots, "int64")
    plain = dev.up(np.full(x.size, 3.0), "float64" if dtype == "float64" else "float32")
    c.read(plain, slots=at)
    wide = dev.down(plain, x.shape)
    for p, seed, offset in ((0.2, 5, 0), (0.5, 6, 1), (0.7, 7, 2 ** 64 - 3), (1.0, 8, 0), (1e-10, 9, 0)):
        out = dev.up(np.full(x.size, 3.0), dtype)
        c.read(out, slots=at, p=p, seed=seed, offset=offset)
        got = dev.down(out, x.shape)
        drop = (ref.dropped(p, seed, offset, x.size) if p < 1 else np.ones(x.size, bool)).reshape(x.shape)
        want = np.where(drop, 0.0, wide / (1 - p) if p < 1 else 0.0)
        want[5] = 3.0
        assert ref.close(got, want, dtype, 2), (p, seed)
        assert np.all(got[5] == 3.0)
    c.close()
    e.close()


# ------------------------------------------------------------------------------------------------ with FromMel and ToMel
@pytest.mark.parametrize("bits,group", [(8, 0), (4, 16)])
def test_to_mel_into_the_cache_and_from_mel_out_of_it(oracle, dev, bits, group):
    """The whole way: waveforms -> ToMel -> cache -> FromMel.  The cached frames are the definition's codes of what ToMel returns, and
    FromMel from the cache is FromMel of what the cache reads as, bit for bit."""
    import gomel_amd
    e = engine(192, GriffinLimIterations=3)
    waves = [oracle.config2_signal(44100, s) for s in (0.5, 0.31, 0.8)]
    mels = e.to_mel_batch(waves)
    counts = [len(m) // 192 for m in mels]
    total = sum(counts)
    c = e.cache(total + 64, bits, group)
    pages = np.random.default_rng(3).permutation(-(-total // 16) + 2) * 16
    slots = (pages[:, None] + np.arange(16)).reshape(-1)[:total].astype(np.int64)
    slots = np.minimum(slots, total + 63)
    assert len(set(slots.tolist())) == total
    assert e.to_mel_cache(waves, c, slots) == counts
    all_pairs = np.concatenate(mels).reshape(total, 192, 2)
    want = ref.stands_for(all_pairs, bits, group)
    got = c.read(np.empty((total, 192, 2)), slots=slots)
    assert ref.close(got, (want, np.abs(want) + 32), "float64", 2)
    at = dev.up(slots, "int64")
    c2 = e.cache(total + 64, bits, group)
    assert e.to_mel_cache(waves, c2, at) == counts                                # slots on the device
    assert np.array_equal(c2.read(np.empty((total, 192, 2)), slots=slots), got)
    cut = np.cumsum([0] + counts)
    per = [slots[a:b] for a, b in zip(cut, cut[1:])]
    outs = e.from_cache(c, per, seeds=[7, 8, 9])
    b = gomel_amd.Batch(e, [k * 192 for k in counts])
    b.upload([got[a:z].reshape(-1, 2) for a, z in zip(cut, cut[1:])], None, [7, 8, 9])
    b.run()
    for o, w in zip(outs, b.download()):
        assert np.array_equal(o, w)
    b.upload_cache(c, at, None, [7, 8, 9])                                        # the same batch again, slots on the device
    b.run()
    for o, w in zip(outs, b.download()):
        assert np.array_equal(o, w)
    # refusals: padding, slots outside, other sizes, another NumMels
    for bad in (-1, total + 64):
        s = slots.copy()
        s[3] = bad
        for where in (s, dev.up(s, "int64")):
            with pytest.raises(gomel_amd.GomelError) as err:
                b.upload_cache(c, where)
            assert err.value.status == 5
    with pytest.raises(gomel_amd.GomelError):
        b.run()                                                                   # not uploaded any more
    assert c.bad_slots() == 0
    b.close()
    with pytest.raises(ValueError):
        e.to_mel_cache(waves, c, slots[:-1])
    s = slots.copy()
    s[0] = total + 64
    with pytest.raises(gomel_amd.GomelError) as err:
        e.to_mel_cache(waves, c, s)
    assert err.value.status == 5
    other = engine(80)
    c80 = other.cache(total)
    with pytest.raises(gomel_amd.GomelError) as err:
        e.to_mel_cache(waves, c80, np.arange(total))
    assert err.value.status == 1
    s = slots.copy()
    s[1], s[2] = -1, s[4]                                                         # padding, and a slot named twice: the later frame
    c.write(np.full((total + 64, 192, 2), 1.5))
    e.to_mel_cache(waves, c, s)
    after = c.read(np.empty((total + 64, 192, 2)))
    assert np.all(after[slots[1]] == 1.5) and np.array_equal(after[slots[4]], got[4]) and np.all(after[slots[2]] == 1.5)
    for k in (c, c2, c80):
        k.close()
    e.close()
    other.close()


@pytest.mark.stress
def test_threads_with_caches_of_their_own_and_a_shared_one(dev):
    """Four threads: staged and device calls on one shared cache (disjoint slots) and on their own."""
    K = 80
    e = engine(K)
    shared = e.cache(400, 8, 0)
    errors = []

    def work(t):
        try:
            own = e.cache(100, 4, 16)
            base = np.arange(100 * t, 100 * t + 100)
            for i in range(6):
                x = frames(100, K, 10 * t + i).astype(np.float32)
                shared.write(x, slots=base)
                own.write(x)
                got = shared.read(np.empty_like(x), slots=base)
                want = ref.stands_for(x.astype(np.float64), 8, 0)
                assert ref.close(got, (want, np.abs(want) + 16), "float32", 1)
                want = ref.stands_for(x.astype(np.float64), 4, 16)
                assert ref.close(own.read(np.empty_like(x)), (want, np.abs(want) + 16), "float32", 1)
                y = e.dropout(x, 0.5, i)
                assert np.array_equal(y == 0, ref.dropped(0.5, i, 0, x.size).reshape(x.shape))
            own.close()
        except Exception as ex:  # noqa: BLE001
            errors.append(repr(ex))

    ts = [threading.Thread(target=work, args=(t,)) for t in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors
    shared.close()
    e.close()


# ------------------------------------------------------------------------------------------------ torch: streams, graphs, autograd
def _torch_child(rep):
    import torch
    rep.stage("torch.cuda init")
    dev = torch.device("cuda", 0)
    torch.zeros(1, device=dev)
    K = 80
    e = engine(K, Device=0)
    c = e.cache(512, 8, 16)

    def want_of(x, bits=8, group=16):
        return ref.stands_for(x.double().cpu().numpy(), bits, group)

    rep.stage("types, strides, alignment")
    for dtype in (torch.float64, torch.float32, torch.float16, torch.bfloat16):
        name = str(dtype).replace("torch.", "")
        for shift in (0, 1, 2, 3, 5):                     # rows that start at any element, in any stride
            wide = torch.randn(33, 2 * K + 7, device=dev).to(dtype)
            x = wide[:, shift:shift + 2 * K].unflatten(1, (K, 2))
            val = torch.empty(33, 2 * K + 3, device=dev, dtype=dtype)
            val.fill_(9)
            v = val[:, 3:].unflatten(1, (K, 2))
            c.write(x, first=100, values=v)
            want = want_of(x)
            assert ref.close(v.double().cpu().numpy(), (want, np.abs(want) + 8), name, 1), (name, shift)
            assert bool((val[:, :3] == 9).all())
            out = torch.full((33, 2 * K + 5), 9, device=dev, dtype=dtype)
            o = out[:, shift:shift + 2 * K].unflatten(1, (K, 2))
            c.read(o, first=100)
            assert torch.equal(o, v), (name, shift)
            assert bool((out[:, :shift] == 9).all()) and bool((out[:, shift + 2 * K:] == 9).all())
            y = e.dropout(wide[:, shift:shift + 2 * K], 0.4, 3, shift)
            drop = ref.dropped(0.4, 3, shift, y.numel()).reshape(y.shape)
            assert ref.close(y.double().cpu().numpy(), np.where(drop, 0, wide[:, shift:shift + 2 * K].double().cpu().numpy() / 0.6), name, 2)
    for bad in (torch.zeros(3, K, 2, device=dev, dtype=torch.int32), torch.zeros(K, 3, 2, device=dev).transpose(0, 1), torch.zeros(3, K, 2)):
        try:
            c.write(bad)
        except ValueError:
            continue
        raise AssertionError("not refused: %s" % bad.dtype)

    rep.stage("large calls")                             # outputs, and rows of the cache, that are stored past the caches
    e192 = engine(192, Device=0)
    for dtype, bits, group, n in ((torch.bfloat16, 8, 64, 120_000), (torch.bfloat16, 8, 0, 350_000), (torch.float64, 4, 32, 40_000), (torch.float32, 8, 16, 320_000),
                                  (torch.float16, 4, 0, 100_000)):
        m = 1000                                         # a thousand frames, again and again: the large call's rows are the small one's
        base = (torch.randn(m, 192, 2, device=dev) * 3).to(dtype)
        small, large = e192.cache(m, bits, group), e192.cache(n, bits, group)
        vs = torch.empty_like(base)
        small.write(base, values=vs)
        x = base.repeat(n // m, 1, 1)
        vl, out, at = torch.empty_like(x), torch.empty_like(x), torch.randperm(n, device=dev)
        large.write(x, slots=at, values=vl)
        large.read(out, slots=at)
        for got in (vl, out):
            assert torch.equal(got.view(n // m, m, 192, 2), vs.expand(n // m, m, 192, 2)), (dtype, bits, group)
        large.read(out, slots=at, p=0.25, seed=3)
        assert torch.equal(out, e192.dropout(vl, 0.25, 3)) or dtype in (torch.float16, torch.bfloat16)
        y = e192.dropout(x, 0.25, 3)
        del large
        wide = torch.empty(n, 390, device=dev, dtype=dtype)
        assert torch.equal(e192.dropout(x.view(n, 384), 0.25, 3, out=wide[:, 3:387]), y.view(n, 384))
        per = 2 ** 20                                    # the dense call against calls of a few MB at their offsets
        for k in (0, x.numel() // per // 2, x.numel() // per - 1):
            part = x.view(-1)[k * per:(k + 1) * per]
            assert torch.equal(y.view(-1)[k * per:(k + 1) * per], e192.dropout(part.clone(), 0.25, 3, offset=k * per)), (dtype, k)
        del x, vl, out, y, wide
    e192.close()

    rep.stage("streams")
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=dev)
    for _ in range(3):
        x = torch.randn(256, K, 2, device=dev)
        out = torch.empty_like(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):                    # the frames are made late on the side stream: the calls have to run behind that
            for _ in range(20):
                big = big @ big
                big = big / big.norm()
            x.mul_(3.0)
            c.write(x, first=0)
            c.read(out, first=0)
            z = e.dropout(out, 0.5, 9)
        side.synchronize()
        want = want_of(x)
        assert ref.close(out.double().cpu().numpy(), (want, np.abs(want) + 30), "float32", 1)
        assert bool(((z == 0) == (torch.from_numpy(ref.dropped(0.5, 9, 0, z.numel())).to(dev).reshape(z.shape) | (out == 0))).all())
    # two writes at once on two streams: neighbouring slots of one cache, both by claims, each naming some of its slots twice
    pair = [torch.cuda.Stream() for _ in range(2)]
    n = 20000
    both = e.cache(2 * n, 8, 16)
    for i in range(4):
        xs = [torch.randn(n, K, 2, device=dev) for _ in range(2)]
        at = [2 * torch.randperm(n, device=dev) + k for k in range(2)]
        for a in at:
            a[: n // 4] = a[n // 4: n // 2]
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(pair[k]):
                both.write(xs[k], slots=at[k])
        torch.cuda.synchronize()
        for k in range(2):
            val, out = torch.empty_like(xs[k]), torch.empty_like(xs[k])
            e.cache(n, 8, 16).write(xs[k], values=val)
            both.read(out, slots=at[k])
            assert torch.equal(out[n // 4:], val[n // 4:]), (i, k)
            assert torch.equal(out[: n // 4], val[n // 4: n // 2]), (i, k)
    both.close()
    s2 = torch.cuda.Stream()
    x = torch.randn(64, K, 2, device=dev)
    torch.cuda.synchronize()
    c.write(x, first=300, stream=s2)                     # a stream named in the call
    s2.synchronize()
    assert ref.close(c.read(np.empty((64, K, 2), np.float32), first=300), (want_of(x), np.abs(want_of(x)) + 8), "float32", 1)

    rep.stage("graphs")
    for n in (32, 2500, 6000):                           # both ways of resolving a slot named twice
        cc = e.cache(8192, 4, 16)
        x, slots = torch.zeros(n, K, 2, device=dev, dtype=torch.bfloat16), torch.zeros(n, dtype=torch.int64, device=dev)
        val, out, drop, back = (torch.zeros_like(x) for _ in range(4))

        def work():
            cc.write(x, slots=slots, values=val)
            cc.read(out, slots=slots)
            cc.read(drop, slots=slots, p=0.25, seed=5)
            e.dropout_backward(val, 0.25, 5, out=back)
        work()
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for g in graphs:                                 # two graphs that share the cache
            with torch.cuda.graph(g):
                work()
        for i in range(6):
            xi = torch.randn(n, K, 2, device=dev).to(torch.bfloat16)
            si = torch.randperm(8192, device=dev)[:n].clone()
            si[n // 2:] = si[:n - n // 2]                # slots named twice
            x.copy_(xi)
            slots.copy_(si)
            graphs[i % 2].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (val, out, drop, back)]
            want = want_of(xi, 4, 16)
            assert ref.close(got[0].double().cpu().numpy(), (want, np.abs(want) + 8), "bfloat16", 1), (n, i)
            last = {int(s): r for r, s in enumerate(si.tolist())}
            rows = torch.tensor([last[int(s)] for s in si.tolist()], device=dev)
            assert torch.equal(got[1], got[0][rows]), (n, i)
            work()                                       # the program's own eager work between the replays
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (val, out, drop, back))), (n, i)
        # a call that would have to stage cannot be captured: refused, and the capture goes on
        import gomel_amd
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            try:
                cc.read(np.empty((2, K, 2), np.float32), stream=torch.cuda.current_stream())
            except gomel_amd.GomelError as ex:
                assert ex.status == 1
            else:
                raise AssertionError("not refused")
            cc.read(out, slots=slots)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got[1])
        cc.close()

    rep.stage("autograd")
    x = torch.randn(37, 2 * K, device=dev, dtype=torch.float64, requires_grad=True)
    y = e.dropout(x, 0.3, 11, 5)
    dy = torch.randn_like(x)
    (dx,) = torch.autograd.grad(y, x, dy)
    keep = ~torch.from_numpy(ref.dropped(0.3, 11, 5, x.numel())).to(dev).reshape(x.shape)
    assert torch.allclose(dx, torch.where(keep, dy / 0.7, torch.zeros_like(dy)), rtol=1e-15, atol=0)
    small = torch.randn(9, device=dev, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: e.dropout(t, 0.4, 2), (small,))
    assert torch.autograd.gradgradcheck(lambda t: e.dropout(t, 0.4, 2), (small,))
    with torch.no_grad():
        out = torch.empty_like(x)
        assert torch.equal(e.dropout(x, 0.3, 11, 5, out=out), y)
    for kw in ({"stream": side}, {"out": torch.empty_like(x)}):
        try:
            e.dropout(x, 0.3, 11, 5, **kw)
        except ValueError:
            continue
        raise AssertionError("not refused")
    # forward and backward captured into a graph, replayed with other inputs, an eager backward between the replays
    xs = torch.randn(64, 161, device=dev, requires_grad=True)
    ds = torch.randn(64, 161, device=dev)
    cap = torch.cuda.Stream()
    cap.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(cap):
        torch.autograd.grad(e.dropout(xs, 0.4, 3), xs, ds)
    torch.cuda.current_stream().wait_stream(cap)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ys = e.dropout(xs, 0.4, 3)
        (gs,) = torch.autograd.grad(ys, xs, ds)
    for i in range(4):
        with torch.no_grad():
            xs.copy_(torch.randn_like(xs))
            ds.copy_(torch.randn_like(ds))
        g.replay()
        torch.cuda.synchronize()
        x2 = xs.detach().clone().requires_grad_(True)
        y2 = e.dropout(x2, 0.4, 3)
        (g2,) = torch.autograd.grad(y2, x2, ds)
        assert torch.equal(ys, y2) and torch.equal(gs, g2), i
    w = torch.randn(2 * K, 64, device=dev, requires_grad=True)       # training from cached frames: cache -> dropout -> a layer -> gradients
    xin = torch.randn(128, K, 2, device=dev)
    c.write(xin, first=0)
    fr = c.read(torch.empty_like(xin), first=0, p=0.1, seed=4).reshape(128, -1)
    h = e.dropout(torch.relu(fr @ w), 0.5, 8)
    h.square().sum().backward()
    frd, wd = fr.double().cpu(), w.detach().double().cpu()
    wd.requires_grad_(True)
    m = torch.from_numpy(~ref.dropped(0.5, 8, 0, 128 * 64)).reshape(128, 64)
    hd = torch.where(m, torch.relu(frd @ wd) / 0.5, torch.zeros(()).double())
    hd.square().sum().backward()
    assert torch.allclose(w.grad.double().cpu(), wd.grad, rtol=1e-3, atol=1e-3 * float(wd.grad.abs().max()))
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_torch_streams_graphs_and_gradients_in_a_child_process():
    import _children
    assert _children.run_child(_torch_child)["ok"]
