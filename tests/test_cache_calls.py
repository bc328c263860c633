"""CPU tests of how the Python side of the spectrogram cache and dropout makes its calls: the stream it picks, what it refuses, what it
counts.  The library is replaced by a recorder; nothing here touches a device."""
import ctypes
import os
import sys
import types

import numpy as np
import pytest

import cache_reference as ref
from test_cache import _Engine, _cache


def _recording(c=None):
    """A cache whose library calls land in a list."""
    c, seen = c or _cache(), []
    c._write = lambda *a: seen.append(a) or 0
    c._read = lambda *a: seen.append(a) or 0
    return c, seen


class _Torch(types.ModuleType):
    """What the choice of a stream asks of torch: cuda.is_initialized, cuda.current_stream(device)."""

    def __init__(self, initialized):
        super().__init__("torch")
        self.cuda = types.SimpleNamespace(is_initialized=lambda: initialized, current_stream=lambda d: types.SimpleNamespace(cuda_stream=0x1000 + d))


@pytest.mark.skipif("torch" in sys.modules, reason="torch is imported: its place is taken")
def test_calls_without_a_tensor_run_on_torchs_current_stream(monkeypatch):
    from gomel_amd import DevicePointer, cache
    c, seen = _recording()
    c.device = 3
    x, d = np.zeros((2, 4, 2)), DevicePointer(4096, 16, "float32")

    def streams():
        del seen[:]
        c.write(x)
        c.read(x, slots=[0, 1])
        c.write(d, slots=DevicePointer(64, 2, "int64"))
        c.read(d)
        c.write(x, stream=7)
        return [a[-1] for a in seen]
    assert streams() == [0, 0, 0, 0, 7]                              # no torch in the process
    monkeypatch.setitem(sys.modules, "torch", _Torch(False))
    assert streams() == [0, 0, 0, 0, 7]                              # torch, but no GPU context of its own
    monkeypatch.setitem(sys.modules, "torch", types.ModuleType("torch"))
    assert streams() == [0, 0, 0, 0, 7]                              # torch half imported
    monkeypatch.setitem(sys.modules, "torch", _Torch(True))
    assert streams() == [0x1003] * 4 + [7]

    class Eng(_Engine):
        class cfg:
            device = 3
            num_mels = 4
    got = []
    cache._dropout(lambda *a: got.append(a[-1]) or 0, "here", Eng, x, 0.5, 1, 0, None, None)
    assert got == [0x1003]
    fake = types.SimpleNamespace(gomel_to_mel_pairs=lambda cfg, n: 4, gomel_to_mel_cache=lambda *a: got.append(a[-1]) or 0,
                                 gomel_batch_upload_cache=lambda *a: got.append(a[-1]) or 0)
    monkeypatch.setattr(cache._lib, "lib", lambda: fake)
    Eng.cfg = ctypes.c_int(0)
    Eng.cfg.num_mels = 4
    assert cache.to_mel_cache(Eng, [np.zeros(9)], c, [1]) == [1]
    batch = types.SimpleNamespace(n_pairs=[4], engine=Eng, _b=None, _x0_args=lambda x0s, seeds: (None, None, None))
    cache.batch_upload_cache(batch, c, [1])
    assert got == [0x1003] * 3


# ------------------------------------------------------------------------------------------------ derivatives (torch, in a child process)
def _derivatives_child(rep):
    """What autograd makes of Engine.dropout, the kernel replaced by its definition in numpy (it sees values only, as the kernel does)."""
    import torch
    import torch.autograd.forward_ad as fwd
    from gomel_amd import cache

    def kernel(fn, where, engine, x, p, seed, offset, out, stream):
        v = x.detach().numpy()
        y = np.where(ref.dropped(p, seed, offset, v.size).reshape(v.shape), 0.0, v / (1 - p))
        return torch.from_numpy(y.astype(v.dtype))
    cache._dropout = kernel
    x, dx, dy = (torch.randn(5, 8, dtype=torch.float64) for _ in range(3))
    for call in (cache.dropout, cache.dropout_backward):
        f = lambda t: call(_Engine, t, 0.4, 11, 3)      # noqa: E731
        want = f(dx)
        with fwd.dual_level():
            y = fwd.unpack_dual(f(fwd.make_dual(x, dx)))
            assert torch.equal(y.primal, f(x)) and y.tangent is not None and torch.equal(y.tangent, want)
            y = fwd.unpack_dual(f(fwd.make_dual(x, dx[:1].expand(5, 8))))          # a tangent that is not dense
            assert torch.equal(y.tangent, f(dx[:1].expand(5, 8).contiguous()))
            assert fwd.unpack_dual(f(x)).tangent is None
            with torch.no_grad():
                assert torch.equal(fwd.unpack_dual(f(fwd.make_dual(x, dx))).tangent, want)
            for kw in ({"out": torch.empty_like(x)}, {"stream": 5}):
                with pytest.raises(ValueError):
                    call(_Engine, fwd.make_dual(x, dx), 0.4, 11, 3, **kw)
        xr = x.clone().requires_grad_(True)
        with fwd.dual_level():                           # both modes at once: the gradient of a directional derivative
            (g,) = torch.autograd.grad((f(fwd.make_dual(xr, dx)) ** 2).sum(), xr)
            t = fwd.unpack_dual(g)
            assert torch.equal(t.primal, 2 * f(f(x))) and torch.equal(t.tangent, 2 * f(f(dx)))
        (g,) = torch.autograd.grad(f(xr), xr, dy)
        assert torch.equal(g, f(dy))
        assert torch.autograd.gradcheck(f, (xr,), check_forward_ad=True, check_batched_grad=False)
    rep.result({"ok": True})


@pytest.mark.torch_child
def test_dropouts_derivatives_in_both_modes():
    import _children
    assert _children.run_child(_derivatives_child)["ok"]


def _tracked_tensors_child(rep):
    """Calls that autograd would have to see, and does not, are refused before anything is written; the rest go through."""
    import torch
    import torch.autograd.forward_ad as fwd
    from gomel_amd import cache
    t = torch.randn(3, 4, 2)
    t.requires_grad_(True)
    plain = torch.randn(3, 4, 2)
    rows = cache._rows

    def taken(a, cols, what, write=False):               # CPU tensors as the GPU's
        return (a.data_ptr(), 1, 8, 3, 0) if cache._is_tensor(a) else rows(a, cols, what, write)
    cache._rows = taken
    cache._stream = lambda stream, device, engine_device: 0
    c, seen = _recording()
    np_out = np.zeros((3, 4, 2), np.float32)
    for frames, values in ((t, plain), (t, t), (plain, t), (t * 2, plain), (plain, t * 2), (t * 2, np_out)):
        with pytest.raises(ValueError, match="gradient"):
            c.write(frames, values=values)
    for out in (t, t * 2):
        with pytest.raises(ValueError, match="gradient"):
            c.read(out)
        with pytest.raises(ValueError, match="gradient"):
            cache.dropout(_Engine, plain, 0.5, 1, out=out)
        with pytest.raises(ValueError, match="gradient"):
            cache.dropout_backward(_Engine, plain, 0.5, 1, out=out)
    with fwd.dual_level():
        d = fwd.make_dual(plain, torch.ones_like(plain))
        for call in (lambda: c.write(d, values=torch.empty(3, 4, 2)), lambda: c.write(t.detach(), values=d), lambda: c.read(d)):
            with pytest.raises(ValueError, match="tangent"):
                call()
    assert seen == []
    c.write(t)                                 # nothing comes back: nothing to differentiate
    c.write(t.detach(), values=plain)
    with torch.no_grad():
        c.write(t, values=plain)
        c.read(t)
    assert len(seen) == 4
    rep.result({"ok": True})


@pytest.mark.torch_child
def test_tensors_that_autograd_follows_are_not_written_behind_its_back():
    import _children
    assert _children.run_child(_tracked_tensors_child)["ok"]


# ------------------------------------------------------------------------------------------------ a runtime call that fails
def test_a_runtime_error_is_a_status():
    """What the cache's and dropout's calls do when the runtime fails: a status and the error's number -- in a child, which must live."""
    import subprocess
    code = ("import ctypes\nfrom gomel_amd import _lib\nL = _lib.lib()\nf = L.gomel_debug_hip_failed\nf.restype, f.argtypes = ctypes.c_int, [ctypes.c_int]\n"
            "assert f(2) == 8 and L.gomel_last_hip_error() == 2\nassert f(719) == 8 and L.gomel_last_hip_error() == 719\nprint('lives')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout == "lives\n", (r.returncode, r.stderr)


# ------------------------------------------------------------------------------------------------ integers of every kind
def test_seeds_and_offsets_are_any_integers():
    from gomel_amd import cache
    c, seen = _recording()
    x = np.zeros((2, 4, 2), np.float32)
    for v, want in ((5, 5), (-1, 2 ** 64 - 1), (2 ** 64 + 3, 3), (np.int64(7), 7), (np.int64(-2), 2 ** 64 - 2), (np.uint32(9), 9), (np.int8(-1), 2 ** 64 - 1),
                    (np.uint64(2 ** 64 - 1), 2 ** 64 - 1), (np.random.default_rng(1).integers(0, 2 ** 40), None), (True, 1)):
        want = int(v) if want is None else want
        del seen[:]
        c.read(x, p=0.5, seed=v, offset=v)
        cache._dropout(lambda *a: seen.append(a) or 0, "here", _Engine, x, 0.5, v, v, None, None)
        for a in seen:
            assert a[-3:-1] == (want, want) and all(type(k) is int for k in a[-3:-1]), v
    for v in (1.0, "1", None, np.float64(2)):
        with pytest.raises(TypeError):
            c.read(x, p=0.5, seed=v)
        with pytest.raises(TypeError):
            c.read(x, p=0.5, offset=v)


def test_numbers_beyond_the_librarys_are_not_cut_off(monkeypatch):
    import gomel_amd
    from gomel_amd import _lib, cache
    c, seen = _recording()
    x = np.zeros((2, 4, 2), np.float32)
    for first in (2 ** 63, 2 ** 64, 2 ** 64 + 3, 2 ** 200):                  # (2 ** 64 + 3 was slot 3)
        del seen[:]
        c.write(x, first=first)
        c.read(x, first=first)
        assert [a[6] for a in seen] == [2 ** 63] * 2                         # no cache has it: the library refuses
    c.write(x, first=np.int64(3))
    assert seen[-1][6] == 3
    with pytest.raises(ValueError):
        c.read(x, first=-2 ** 70)
    L, made = _lib.lib(), []
    cfg = _lib.GomelConfig()
    L.gomel_default_config(ctypes.byref(cfg))
    eng = types.SimpleNamespace(cfg=cfg, _h=None)
    monkeypatch.setattr(cache._lib, "lib", lambda: types.SimpleNamespace(gomel_cache_frame_bytes=L.gomel_cache_frame_bytes, gomel_cache_write=None, gomel_cache_read=None,
                                                                         gomel_cache_create=lambda h, n, b, g, out: made.append((n, b, g)) or 0,
                                                                         gomel_cache_destroy=lambda c: 0))
    for args, want in (((2 ** 64 + 4, 8, 0), (2 ** 63, 8, 0)), ((4, 2 ** 32 + 8, 0), (4, -1, 0)), ((4, 8, 2 ** 32), (4, 8, -1)), ((4, 8 - 2 ** 32, 16), (4, -1, 16)),
                       ((5, 4, 64), (5, 4, 64))):
        k = gomel_amd.Cache(eng, *args)
        assert made.pop() == want and (k.frame_bytes > 0) == (want[1] > 0 and want[2] >= 0)


# ------------------------------------------------------------------------------------------------ the slots of several utterances
def test_slots_of_several_utterances():
    from gomel_amd import DevicePointer
    from gomel_amd.cache import _joined
    for slots in ([[1, 2, 3], [4, 5]], [np.array([1, 2, 3], np.int32), (4, 5)], [np.array([[1], [2], [3]]), np.uint64([4, 5])]):
        flat, counts = _joined(slots, None, 0)
        assert flat.dtype == np.int64 and flat.tolist() == [1, 2, 3, 4, 5] and counts == [3, 2]
    p = DevicePointer(64, 7, "int64")
    assert _joined([p], None, 0) == (p, [7])
    for slots in ([[1.0, 2.5]], [np.array([1.0])], [[1], [2 ** 63]], [["1"]], [p, p], [p, [1]], [np.array([2 ** 63], np.uint64)]):
        with pytest.raises(ValueError):
            _joined(slots, None, 0)


def test_from_cache_refuses_before_it_allocates_a_batch(monkeypatch):
    from gomel_amd import DevicePointer, cache
    c = _cache()

    def batch(*a):
        raise AssertionError("a batch was allocated")
    monkeypatch.setattr(cache, "Batch", batch)
    assert cache.from_cache(_Engine, c, []) == [] and cache.from_cache(_Engine, c, iter(())) == []
    p = DevicePointer(64, 7, "int64")
    for slots in ([[1.5]], [p, p], [[1], p], iter([[1], [0.5]])):
        with pytest.raises(ValueError):
            cache.from_cache(_Engine, c, slots)


# ------------------------------------------------------------------------------------------------ closed or collected in a capture
def test_a_cache_dropped_in_a_capture_is_destroyed_behind_it(monkeypatch):
    import gc
    from gomel_amd import cache
    gone, busy = [], [True]
    monkeypatch.setattr(cache, "_left", [])
    monkeypatch.setattr(cache, "_capturing", lambda stream, device: busy[0])
    monkeypatch.setattr(cache._lib, "lib", lambda: types.SimpleNamespace(gomel_cache_destroy=lambda c: gone.append(c.value) or 0))

    def made(v):
        c, _ = _recording()
        c._c = ctypes.c_void_p(v)
        return c
    a, b, live = made(11), made(12), made(13)
    x = np.zeros((1, 4, 2), np.float32)
    a.close()
    a.close()
    del b
    gc.collect()
    live.write(x)
    live.read(x)
    assert gone == []                                    # the capture goes on
    busy[0] = False
    live.read(x)
    assert sorted(gone) == [11, 12]
    made(14).close()
    busy[0] = True
    made(15).close()
    assert sorted(gone) == [11, 12, 14]
    busy[0] = False
    live.close()
    assert sorted(gone) == [11, 12, 13, 14, 15]


def test_calls_that_wait_are_refused_in_a_capture(monkeypatch):
    import gomel_amd
    from gomel_amd import cache
    monkeypatch.setattr(cache, "_capturing", lambda stream, device: True)
    c, _ = _recording()
    c._c = ctypes.c_void_p(1)
    try:
        for call in (c.bad_slots, lambda: gomel_amd.Cache(_Engine, 4), lambda: cache.from_cache(_Engine, c, [[1]])):
            with pytest.raises(gomel_amd.GomelError) as err:
                call()
            assert err.value.status == 1
    finally:
        c._c = ctypes.c_void_p()


# ------------------------------------------------------------------------------------------------ how far a value reads from what was written
def bound(x, lo, step, hi, dtype):
    """include/gomel_hip.h's bound before the read's rounding, x [..] float64 values of one group each (lo, step, hi broadcast to them)."""
    b = step.astype(np.float64) / 2 + np.where(step < 2.0 ** -126, 2.0 ** -142, 0.0)
    if dtype == "float64":
        b = b + 2.0 ** -24 * np.maximum(np.abs(lo.astype(np.float64)), np.abs(hi)) + 2.0 ** -150
    return b * (1 + 2.0 ** -40)                          # the definition's own fp64 arithmetic


def hard_groups(rng, n, K, dtype):
    """Frames of every size and offset: spans from subnormal to the whole range, offsets far above the span, equal values."""
    top = {"float64": 38, "float32": 38, "float16": 4, "bfloat16": 38}[dtype]
    span = 10.0 ** rng.uniform(-44 if dtype != "float16" else -7, top, (n, 1, 1))
    off = rng.choice([0.0, 1.0, 1e3, 1e-3], (n, 1, 1)) * span * rng.uniform(-2, 2, (n, 1, 1))
    x = off + span * rng.random((n, K, 2)) * rng.choice([1.0, 1.0, 1e-6, 0.0], (n, 1, 1))
    big = {"float64": 3.4e38, "float32": 3.4e38, "float16": 65504.0, "bfloat16": 3.38e38}[dtype]
    return np.clip(x, -big, big)


@pytest.mark.parametrize("dtype", ["float64", "float32", "float16", "bfloat16"])
def test_the_contracts_bound(dtype):
    rng = np.random.default_rng(12)
    x = hard_groups(rng, 1500, 16, dtype)
    x[:3] = [[1.0, 1.0 + 1e-9]], [[1000.0, 1000.001]], [[0.0, 370 * 2.0 ** -149]]
    x = (ref.from_bf16(ref.to_bf16(x.astype(np.float32))) if dtype == "bfloat16" else x.astype(dtype)).astype(np.float64)
    for bits in (8, 4):
        for group in (0, 8):
            q, lo, step = ref.quantise(x, bits, group)
            of = np.arange(16) // (group or 16)
            hi = x.reshape(len(x), -1, group or 16, 2).max((2, 3))
            off = np.abs(ref.stands_for(x, bits, group) - x)
            b = bound(x, lo[:, of, None], step[:, of, None], hi[:, of, None], dtype)
            # stands_for's own sum: two roundings of 2^-53 of its larger operand
            assert np.all(off <= b + 2.0 ** -52 * (np.abs(lo[:, of, None]) + 16 * np.abs(x))), (bits, group, np.max(off / np.maximum(b, 1e-300)))
            if dtype in ("float64", "float32"):
                assert np.any(off > step[:, of, None] * 0.51)         # half a step alone does not hold


# ------------------------------------------------------------------------------------------------ the first tensor of a process
def _first_tensor_child(rep):
    import torch
    from gomel_amd import cache
    with torch.inference_mode():
        t = torch.zeros(3, 4, 2)
        assert cache._is_tensor(t)
        cache._written(t)                                # has no version to count
    u = torch.zeros(3)
    cache._written(u)
    assert u._version == 1
    rep.result({"ok": True})


@pytest.mark.torch_child
def test_the_first_tensor_may_be_an_inference_tensor():
    import _children
    assert _children.run_child(_first_tensor_child)["ok"]
