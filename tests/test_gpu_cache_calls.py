"""GPU tests of how the spectrogram cache and dropout are called: streams, captures, derivatives, calls that fail on the way.  Values are
held against the definitions (cache_reference.py) or against the same call made one step at a time; what a kernel computes is
test_gpu_cache.py's subject."""
import ctypes

import numpy as np
import pytest

import cache_reference as ref
from test_cache_calls import bound, hard_groups
from test_gpu_cache import TYPES, dev, engine, frames, held  # noqa: F401  (dev: the fixture)

pytestmark = [pytest.mark.gpu]


def _late(torch, stream, n=20):
    """Work of some milliseconds on `stream`: whatever is queued there behind it happens late."""
    with torch.cuda.stream(stream):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(n):
            big = big @ big
            big = big / big.norm()


# ------------------------------------------------------------------------------------------------ slots made late on a named stream
def _from_cache_child(rep):
    import torch
    rep.stage("torch.cuda init")
    torch.zeros(1, device="cuda")
    e = engine(16, Device=0, GriffinLimIterations=2)
    c = e.cache(64, 8, 0)
    x = torch.randn(64, 16, 2, device="cuda")
    c.write(x)
    side = torch.cuda.Stream()
    want = e.from_cache(c, [np.arange(8, 20), np.arange(30, 45)], seeds=[1, 2])
    rep.stage("slots written late on the stream that the call names")
    for named in (side, side.cuda_stream):
        at = [torch.zeros(12, dtype=torch.int64, device="cuda"), torch.zeros(15, dtype=torch.int64, device="cuda")]   # slot 0 until then
        first = [torch.arange(8, 20, device="cuda"), torch.arange(30, 45, device="cuda")]
        torch.cuda.synchronize()
        _late(torch, side)
        with torch.cuda.stream(side):
            for a, f in zip(at, first):
                a.copy_(f)
        got = e.from_cache(c, at, seeds=[1, 2], stream=named)
        assert all(np.array_equal(g, w) for g, w in zip(got, want))
    rep.stage("the stream named, the current one busy")
    torch.cuda.synchronize()
    _late(torch, torch.cuda.current_stream())
    got = e.from_cache(c, first, seeds=[1, 2], stream=side)
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    got = e.from_cache(c, first, seeds=[1, 2], stream=0)
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    rep.stage("no stream named: the current one")
    at = [torch.zeros(12, dtype=torch.int64, device="cuda"), torch.zeros(15, dtype=torch.int64, device="cuda")]
    torch.cuda.synchronize()
    _late(torch, side)
    with torch.cuda.stream(side):
        for a, f in zip(at, first):
            a.copy_(f)
        got = e.from_cache(c, at, seeds=[1, 2])
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_from_cache_joins_its_slots_on_the_stream_of_the_call():
    import _children
    assert _children.run_child(_from_cache_child)["ok"]


# ------------------------------------------------------------------------------------------------ an engine whose configuration names no device
def test_an_engine_knows_its_device():
    import gomel_amd
    from gomel_amd import _lib
    m = gomel_amd.NewMel()
    assert m.Device == -1
    cfg = m._config()
    e = gomel_amd.Engine(cfg)
    assert cfg.device == -1 and e.cfg.device == 0 == _lib.lib().gomel_device(e._h) and e.cache(4).device == 0
    e.close()


def _vouched_child(rep):
    import torch
    torch.zeros(1, device="cuda")
    import gomel_amd.cache as gc
    e = engine(16)                                       # Device = -1
    c = e.cache(8)
    seen = []
    write, read = c._write, c._read
    c._write, c._read = (lambda *a: seen.append(a[1]) or write(*a)), (lambda *a: seen.append(a[1]) or read(*a))
    x, at = torch.randn(3, 16, 2, device="cuda"), torch.arange(3, device="cuda")
    v, out = torch.empty_like(x), torch.empty_like(x)
    c.write(x, slots=at, values=v)
    c.read(out, slots=at)
    assert seen == [1 | gc._ON_DEVICE] * 2 and torch.equal(v, out)
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_an_engine_without_a_named_device_vouches_for_its_tensors():
    import _children
    assert _children.run_child(_vouched_child)["ok"]


# ------------------------------------------------------------------------------------------------ calls without a tensor follow the tensor calls
def _no_tensor_child(rep):
    import torch
    import gomel_amd
    rep.stage("torch.cuda init")
    torch.zeros(1, device="cuda")
    K = 16
    e = engine(K, Device=0, GriffinLimIterations=2)
    side = torch.cuda.Stream()
    x = torch.randn(64, K, 2, device="cuda")
    c, c2 = e.cache(64, 8, 0), e.cache(64, 8, 0)
    c2.write(x)
    want = c2.read(np.empty((64, K, 2), np.float32))
    waves = e.from_cache(c2, [np.arange(10, 30)], seeds=[5])
    out = torch.zeros(64, K, 2, device="cuda")
    for what in ("read", "from_cache", "DevicePointer", "dropout"):
        rep.stage(what)
        c.write(torch.zeros_like(x))
        out.zero_()
        torch.cuda.synchronize()
        _late(torch, side)
        with torch.cuda.stream(side):
            c.write(x)                                   # late: on the side stream, behind its work
            if what == "read":
                assert np.array_equal(c.read(np.empty((64, K, 2), np.float32)), want)
            elif what == "from_cache":
                assert np.array_equal(e.from_cache(c, [list(range(10, 30))], seeds=[5])[0], waves[0])
            elif what == "DevicePointer":
                c.read(gomel_amd.DevicePointer(out.data_ptr(), out.numel(), "float32"))
                side.synchronize()
                assert np.array_equal(out.cpu().numpy(), want)
            else:
                c.read(out)
                y = gomel_amd.DevicePointer(out.data_ptr(), out.numel(), "float32")
                e.dropout(y, 1.0, 3, out=y)
                side.synchronize()
                assert not out.any()
    rep.stage("to_mel_cache: a tensor read queued before it sees what was there before it")
    wave = np.random.default_rng(0).normal(size=30000)
    n = e.to_mel_cache([wave], c, np.arange(len(e.to_mel_batch([wave])[0]) // K))[0]
    c.write(x)
    torch.cuda.synchronize()
    _late(torch, side)
    with torch.cuda.stream(side):
        c.read(out)
        e.to_mel_cache([wave], c, list(range(n)))
        side.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    for k in (c, c2):
        k.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_calls_without_a_tensor_follow_the_current_stream():
    import _children
    assert _children.run_child(_no_tensor_child)["ok"]


# ------------------------------------------------------------------------------------------------ derivatives
def _forward_mode_child(rep):
    import torch
    import torch.autograd.forward_ad as fwd
    torch.zeros(1, device="cuda")
    e = engine(16, Device=0)
    x, dx = (torch.randn(33, 7, device="cuda", dtype=torch.float64) for _ in range(2))
    with fwd.dual_level():
        y = fwd.unpack_dual(e.dropout(fwd.make_dual(x, dx), 0.3, 5, 2))
        assert torch.equal(y.primal, e.dropout(x, 0.3, 5, 2)) and torch.equal(y.tangent, e.dropout(dx, 0.3, 5, 2))
        y = fwd.unpack_dual(e.dropout_backward(fwd.make_dual(x, dx), 0.3, 5, 2))
        assert torch.equal(y.tangent, e.dropout(dx, 0.3, 5, 2))
    small = torch.randn(11, device="cuda", dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: e.dropout(t, 0.4, 2), (small,), check_forward_ad=True)
    e.close()
    rep.result({"ok": True})


def _versions_child(rep):
    """A buffer that autograd holds for a backward pass and a call then writes to: that pass raises, as after torch's own in-place writes."""
    import torch
    torch.zeros(1, device="cuda")
    e = engine(16, Device=0)
    c = e.cache(8)
    w = torch.randn(16, 2, device="cuda", requires_grad=True)
    c.write(torch.randn(3, 16, 2, device="cuda"))
    for write in (lambda b: c.read(b), lambda b: c.read(b, p=0.5, seed=1), lambda b: c.write(torch.randn_like(b), values=b), lambda b: c.write(b, values=b),
                  lambda b: e.dropout(torch.randn_like(b), 0.5, 1, out=b), lambda b: e.dropout_backward(b, 0.5, 1, out=b),
                  lambda b: e.dropout(torch.randn_like(b), 0.5, 1, out=b, stream=torch.cuda.current_stream()),
                  lambda b: c.read(b.view(3, 32).view(3, 16, 2))):
        buf = torch.randn(3, 16, 2, device="cuda")
        loss = (w * buf).sum()                               # the product holds buf
        write(buf)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
    buf = torch.randn(3, 16, 2, device="cuda")
    loss = (w * buf).sum()
    c.write(buf)                                             # only read: nothing to tell
    e.dropout(buf, 0.5, 1)
    loss.backward()
    with torch.inference_mode():                             # tensors without a version
        buf = torch.randn(3, 16, 2, device="cuda")
        c.read(buf)
        c.write(buf, values=buf)
        e.dropout(buf, 0.5, 1, out=buf)
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_autograd_sees_what_a_call_has_written():
    import _children
    assert _children.run_child(_versions_child)["ok"]


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_dropout_in_forward_mode():
    import _children
    assert _children.run_child(_forward_mode_child)["ok"]


# ------------------------------------------------------------------------------------------------ tensors dropped while a named stream uses them
def _dropped_tensors_child(rep):
    import torch
    torch.zeros(1, device="cuda")
    K, n = 80, 3000
    e = engine(K, Device=0)
    c = e.cache(n)
    base = torch.randn(n, K, 2, device="cuda", dtype=torch.float64)
    at = torch.randperm(n, device="cuda", dtype=torch.int64)
    want, y_want = torch.empty(n, K, 2, device="cuda"), torch.empty(n, K, 2, device="cuda")
    c.write(base.float(), values=want)
    e.dropout(base.float(), 0.5, 1, out=y_want)
    side = torch.cuda.Stream()

    def others(*like):                                   # memory of these sizes, freed just now, goes to somebody else at once
        return [torch.full_like(t, 7) for t in like for _ in range(3)]
    for named in (side, side.cuda_stream):
        c.write(torch.zeros_like(want))
        out, y, val = (torch.empty_like(want) for _ in range(3))
        like, like_at = torch.empty_like(want), torch.empty_like(at)
        torch.cuda.synchronize()
        _late(torch, side)
        x, x2, at1, at2 = base.float(), base.float(), at.clone(), at.clone()
        side.wait_stream(torch.cuda.current_stream())
        c.write(x, slots=at1, values=val, stream=named)
        c.read(out, slots=at2, stream=named)
        e.dropout(x2, 0.5, 1, out=y, stream=named)
        del x, x2, at1, at2
        held = others(like, like_at)
        c.read(torch.empty_like(out), stream=named)      # an output that nobody keeps: it must not be written over somebody else's memory
        held += others(like)
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(val, want) and torch.equal(y, y_want)
        assert all(bool((h == 7).all()) for h in held)
        del held
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_tensors_dropped_while_a_named_stream_uses_them():
    import _children
    assert _children.run_child(_dropped_tensors_child)["ok"]


# ------------------------------------------------------------------------------------------------ calls that wait, in a capture
def _capture_child(rep):
    import torch
    import gomel_amd
    torch.zeros(1, device="cuda")
    K = 16
    e = engine(K, Device=0, GriffinLimIterations=2)
    c = e.cache(64)
    x, out = torch.randn(40, K, 2, device="cuda"), torch.empty(40, K, 2, device="cuda")
    c.write(x)
    at = torch.arange(5, 25, device="cuda")
    wave = np.random.default_rng(0).normal(size=30000)
    n = len(e.to_mel_batch([wave])[0]) // K
    b = gomel_amd.Batch(e, [20 * K])
    want = e.from_cache(c, [at], seeds=[3])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.write(x)
        named = torch.cuda.current_stream()
        for call in (lambda: e.from_cache(c, [at], seeds=[3]), lambda: e.from_cache(c, [list(range(5, 25))], seeds=[3]),
                     lambda: e.from_cache(c, [list(range(5, 25))], seeds=[3], stream=named.cuda_stream),
                     lambda: b.upload_cache(c, at), lambda: b.upload_cache(c, np.arange(20)), lambda: b.upload_cache(c, at, stream=named),
                     lambda: e.to_mel_cache([wave], c, list(range(n))), lambda: e.to_mel_cache([wave], c, list(range(n)), stream=named),
                     c.bad_slots, lambda: e.cache(4)):
            with pytest.raises(gomel_amd.GomelError) as err:
                call()
            assert err.value.status == 1
        c.read(out)
    for i in range(3):
        xi = torch.randn_like(x)
        x.copy_(xi)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        c.write(xi, values=out)                          # the program's own work between the replays
        assert torch.equal(got, out), i
        assert e.to_mel_cache([wave], c, list(range(n))) == [n]
        b.upload_cache(c, at, None, [3])
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    c.write(x, values=out)
    assert not np.array_equal(e.from_cache(c, [at], seeds=[3])[0], want[0])
    b.close()
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_calls_that_wait_are_refused_in_a_capture_which_goes_on():
    import _children
    assert _children.run_child(_capture_child)["ok"]


# ------------------------------------------------------------------------------------------------ a runtime call that fails
def test_a_cache_that_does_not_fit_the_memory():
    import gomel_amd
    from gomel_amd import _lib
    e = engine(80)
    with pytest.raises(gomel_amd.GomelError) as err:
        e.cache(2 ** 36)                                 # 12 TB
    assert err.value.status == 8 and _lib.lib().gomel_last_hip_error() == 2
    c = e.cache(4)                                       # and everything goes on
    x = frames(4, 80, 1).astype(np.float32)
    c.write(x)
    assert np.any(c.read(np.empty_like(x)) != 0)
    c.close()
    e.close()


# ------------------------------------------------------------------------------------------------ a launch that fails
@pytest.mark.parametrize("K,dtype,group,n", [(24, "float32", 8, 5000), (515, "float64", 0, 2100), (515, "float64", 32, 4200)])
def test_a_write_that_fails_leaves_no_claim_behind(dev, K, dtype, group, n):  # noqa: F811
    """The frames claim their slots in a launch before the write's.  When the write's fails, the next write of the same slots from other,
    lower rows has to reach the cache: frames under one scale, in segments and block-wide."""
    import gomel_amd
    from gomel_amd import _lib
    e = engine(K, Resolut=8192) if K > 700 else engine(K)
    c = e.cache(n, 8, group)
    x = frames(8, K, 1)
    want = ref.stands_for(held(x, dtype), 8, group)
    which = np.arange(n) % 8
    src, up, down = dev.up(x[which], dtype), dev.up(np.arange(n), "int64"), dev.up(np.arange(n)[::-1], "int64")
    fail = _lib.lib().gomel_debug_fail_launch
    fail.restype, fail.argtypes = None, [ctypes.c_int]
    fail(1)
    with pytest.raises(gomel_amd.GomelError) as err:
        c.write(src, slots=up)
    assert err.value.status == 8
    assert not c.read(np.empty((n, K, 2))).any()
    c.write(src, slots=down)                             # slot n - 1 now comes from row 0: a claim of row n - 1 must not stand in its way
    got = c.read(np.empty((n, K, 2)))[::-1]
    for i in range(8):
        assert ref.close(got[which == i], (np.broadcast_to(want[i], got[which == i].shape), np.abs(want[i]) + 32), "float64", 2), i
    c.write(src, slots=up)
    assert np.array_equal(c.read(np.empty((n, K, 2))), got)
    c.close()
    e.close()


# ------------------------------------------------------------------------------------------------ the slots of several utterances
def test_slots_of_every_kind_into_from_mel(dev):  # noqa: F811
    K = 16
    e = engine(K, GriffinLimIterations=2)
    c = e.cache(64)
    c.write(frames(64, K, 2))
    want = e.from_cache(c, [np.arange(8, 20), np.arange(30, 45)], seeds=[1, 2])
    for slots in ([list(range(8, 20)), tuple(range(30, 45))], [np.arange(8, 20)[:, None], np.arange(30, 45, dtype=np.uint8)], iter([range(8, 20), range(30, 45)])):
        got = e.from_cache(c, slots, seeds=[1, 2])
        assert all(np.array_equal(g, w) for g, w in zip(got, want)) and len(got) == 2
    assert np.array_equal(e.from_cache(c, [dev.up(np.arange(8, 20), "int64")], seeds=[1])[0], want[0])
    c.close()
    e.close()


def _slot_tensors_child(rep):
    import torch
    torch.zeros(1, device="cuda")
    e = engine(16, Device=0, GriffinLimIterations=2)
    c = e.cache(64)
    a, b = torch.arange(8, 20, device="cuda"), torch.arange(30, 45, device="cuda")
    c.write(torch.randn(64, 16, 2, device="cuda"))
    want = e.from_cache(c, [a, b], seeds=[1, 2])
    got = e.from_cache(c, [a.view(3, 4), torch.arange(30, 60, device="cuda")[:30].view(15, 2)[:, 0] * 0 + b], seeds=[1, 2])
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    for bad in ([a, [30, 31]], [a, b.int()], [a.float(), b], [a, b.cpu()], [a.cpu()], [a > 3]):
        with pytest.raises(ValueError):
            e.from_cache(c, bad)
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_slot_tensors_into_from_mel():
    import _children
    assert _children.run_child(_slot_tensors_child)["ok"]


# ------------------------------------------------------------------------------------------------ closed or collected in a capture
def _dropped_in_a_capture_child(rep):
    import gc
    import torch
    torch.zeros(1, device="cuda")
    K = 16
    e = engine(K, Device=0)
    c = e.cache(64)
    x, out = torch.randn(64, K, 2, device="cuda"), torch.empty(64, K, 2, device="cuda")
    free0 = torch.cuda.mem_get_info()[0]
    big, other = e.cache(2 ** 26), e.cache(2 ** 25)      # 3.5 and 1.7 GB
    held = [big]
    held.append(held)                                    # a cycle: the collector finds it
    c.write(x)
    torch.cuda.synchronize()
    assert free0 - torch.cuda.mem_get_info()[0] > 4 << 30
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.write(x)
        del big, held
        gc.collect()
        other.close()
        c.read(out)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        c.write(x, values=out)
        assert torch.equal(got, out), i
    torch.cuda.synchronize()
    assert free0 - torch.cuda.mem_get_info()[0] < 1 << 30
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_caches_dropped_in_a_capture_leave_it_alone():
    import _children
    assert _children.run_child(_dropped_in_a_capture_child)["ok"]


# ------------------------------------------------------------------------------------------------ beside a persistent launch
def test_from_mel_out_of_the_cache_waits_for_a_persistent_launch():
    """The read of upload_cache is ordinary kernel work: it goes behind a persistent run of another engine, not beside it."""
    import time
    import gomel_amd
    K = 80
    one = engine(K, Resolut=1024, Window=256, MelFmax=8000, GriffinLimIterations=4000)
    one.set_path(3)                                      # persistent
    one.set_precision(32)
    other = engine(K)
    c = other.cache(64)
    c.write(frames(64, K, 1))
    b, run = gomel_amd.Batch(other, [40 * K]), gomel_amd.Batch(one, [40 * K])
    run.upload([frames(40, K, 3).reshape(-1, 2)], None, [1])
    assert run.run_timed()["fast_path"] == 2
    b.upload_cache(c, np.arange(40))
    left = []
    for _ in range(3):
        t0 = time.perf_counter()
        run.run()
        b.upload_cache(c, np.arange(40))
        t1 = time.perf_counter()
        run.sync()
        t2 = time.perf_counter()
        assert t2 - t0 > 0.01, "the run is too short to show the order"
        left.append((t2 - t1) / (t2 - t0))               # of the run, when the upload was through (0.99 beside it)
    assert min(left) < 0.2, left
    for k in (b, run, c, one, other):
        k.close()


# ------------------------------------------------------------------------------------------------ bad slots counted beside running calls
def _bad_slots_child(rep):
    import torch
    torch.zeros(1, device="cuda")
    K, n, rounds = 16, 200_000, 400
    e = engine(K, Device=0)
    c = e.cache(64)
    out = torch.zeros(n, K, 2, device="cuda")
    at = torch.full((n,), 64, device="cuda")             # every one beyond the cache
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    told, mid = 0, 0
    with torch.cuda.stream(side):
        for _ in range(rounds):
            c.read(out, slots=at)
            told += c.bad_slots()
            mid += 0 < told < n * rounds
    side.synchronize()
    told += c.bad_slots()
    assert told == n * rounds and c.bad_slots() == 0 and mid > 0, (told, n * rounds, mid)
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_no_bad_slot_is_lost_to_a_count_beside_a_running_call():
    import _children
    assert _children.run_child(_bad_slots_child)["ok"]


# ------------------------------------------------------------------------------------------------ how far a value reads from what was written
@pytest.mark.parametrize("dtype", TYPES)
def test_reads_keep_the_contracts_bound(dev, dtype):  # noqa: F811
    """Bound of include/gomel_hip.h with the read's rounding, for the type that was written and for float64."""
    K, n = 16, 1500
    e = engine(K)
    x = held(hard_groups(np.random.default_rng(5), n, K, dtype), dtype)
    for bits, group in ((8, 0), (4, 8)):
        c = e.cache(n, bits, group)
        c.write(dev.up(x, dtype))
        _, lo, step = ref.quantise(x, bits, group)
        of = np.arange(K) // (group or K)
        hi = x.reshape(n, -1, group or K, 2).max((2, 3))
        b = bound(x, lo[:, of, None], step[:, of, None], hi[:, of, None], dtype)
        for out_type in {dtype, "float64"}:
            out = dev.empty(x.size, out_type)
            c.read(out)
            got = dev.down(out, x.shape)
            v = np.abs(x) + b
            wide = 2.0 ** -53 if out_type == "float64" else 2.0 ** -24
            room = v * wide * 1.001 + (v * ref.HALF[out_type] * 1.001 if out_type in ("float16", "bfloat16") else 0) + 2 * ref.TINY[out_type] + 2 * ref.TINY["float32"]
            fits = v < {"float64": 1e300, "float32": 3.4e38, "float16": 65000.0, "bfloat16": 3.38e38}[out_type]
            assert np.all(np.abs(got - x)[fits] <= (b + room)[fits]), (bits, group, out_type)
        c.close()
    e.close()


# ------------------------------------------------------------------------------------------------ forms that other sizes do not reach
@pytest.mark.parametrize("K,dtype", [(350, "float64"), (700, "float32"), (1400, "float16"), (1400, "bfloat16"), (161, "float64"), (383, "float64")])
def test_rows_of_up_to_six_units_a_lane(dev, K, dtype):  # noqa: F811
    """Rows of 321 ... 384 units of 16 bytes (six to each of 64 lanes), one scale a frame and groups, few frames and many; and their
    neighbours of 3 and 6 units with a last one that is partial or missing."""
    e = engine(K, Resolut=8192) if K > 700 else engine(K)
    for bits, group in ((8, 0), (4, 0), (8, 16), (4, 64)):
        for n in (5, 4500):                              # at most 4096: a wave for a frame
            base = frames(8, K, K + n)
            xd = held(base, dtype)
            want, (q, lo, step) = ref.stands_for(xd, bits, group), ref.quantise(xd, bits, group)
            of = np.arange(K) // (group or K)
            size = np.abs(lo)[:, of, None] + q * step[:, of, None].astype(np.float64)
            c = e.cache(n, bits, group)
            which, slots = np.arange(n) % 8, np.random.default_rng(n).permutation(n).astype(np.int64)
            src, val, out, at = dev.up(base[which], dtype), dev.empty(n * 2 * K, dtype), dev.empty(n * 2 * K, dtype), dev.up(slots, "int64")
            c.write(src, slots=at, values=val)
            c.read(out, slots=at)
            got, back = dev.down(out, (n, K, 2)), dev.down(val, (n, K, 2))
            assert np.array_equal(got, back), (bits, group, n)
            for i in range(min(n, 8)):
                assert ref.close(got[i], (want[i], size[i]), dtype, 1), (bits, group, n, i)
                assert np.array_equal(got[which == i], np.broadcast_to(got[i], got[which == i].shape)), (bits, group, n, i)
            c.close()
    e.close()


def _large_read_with_dropout_child(rep):
    """Outputs of 64 MB and more with dropout: bit for bit what small reads give, each at the counter of its first element."""
    import torch
    torch.zeros(1, device="cuda")
    K = 192
    e = engine(K, Device=0)
    for dtype in (torch.float16, torch.bfloat16, torch.float32, torch.float64):
        n = (64 << 20) // (2 * K * torch.empty(0, dtype=dtype).element_size()) + 1003
        for bits, group in ((8, 0), (4, 32)):
            c = e.cache(n, bits, group)
            at = torch.randperm(n, device="cuda")
            c.write((torch.randn(n, K, 2, device="cuda") * 3).to(dtype))
            large, plain = torch.empty(n, K, 2, device="cuda", dtype=dtype), torch.empty(n, K, 2, device="cuda", dtype=torch.float64 if dtype == torch.float64 else torch.float32)
            for p, seed, offset in ((0.25, 3, 0), (0.6, 2 ** 63 + 1, 7)):
                c.read(large, slots=at, p=p, seed=seed, offset=offset)
                small = torch.empty_like(large)
                step = 9000
                for r in range(0, n, step):
                    c.read(small[r:r + step], slots=at[r:r + step], p=p, seed=seed, offset=offset + 2 * K * r)
                assert torch.equal(large, small), (dtype, bits, group, p)
                # against the definition: dropout of the wide read, rounded once
                c.read(plain, slots=at)
                for r in (0, n // 2, n - 40):
                    drop = ref.dropped(p, seed, offset + 2 * K * r, 40 * 2 * K).reshape(40, K, 2)
                    want = np.where(drop, 0.0, plain[r:r + 40].double().cpu().numpy() / (1 - p))
                    assert ref.close(large[r:r + 40].double().cpu().numpy(), want, str(dtype).replace("torch.", ""), 2), (dtype, bits, group, p, r)
            c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_large_reads_with_dropout_in_every_type():
    import _children
    assert _children.run_child(_large_read_with_dropout_child)["ok"]


# ------------------------------------------------------------------------------------------------ streams that are not torch's
def _foreign_stream_child(rep):
    """A call on a stream that the program makes and ends by itself, before the tensors go."""
    import torch
    import gomel_amd
    torch.zeros(1, device="cuda")
    hip = ctypes.CDLL(gomel_amd.hip_runtime_path())
    hip.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    hip.hipStreamSynchronize.argtypes = hip.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    e = engine(80, Device=0)
    c = e.cache(500)
    x, at = torch.randn(500, 80, 2, device="cuda"), torch.randperm(500, device="cuda")
    want, y_want = torch.empty_like(x), torch.empty_like(x)
    c.write(x, slots=at, values=want)
    e.dropout(x, 0.5, 1, out=y_want)
    for kind in (int, lambda h: torch.cuda.ExternalStream(h)):
        s = ctypes.c_void_p()
        assert hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
        out, val, y, at2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), at.clone()
        torch.cuda.synchronize()
        named = kind(s.value)
        c.write(x, slots=at2, values=val, stream=named)
        c.read(out, slots=at2, stream=named)
        e.dropout(x, 0.5, 1, out=y, stream=named)
        del at2
        torch.full_like(at, 3)                           # torch's stream is behind the calls: no wait is needed to reuse or to read
        assert torch.equal(out, want) and torch.equal(val, want) and torch.equal(y, y_want)
        assert hip.hipStreamSynchronize(s) == 0 and hip.hipStreamDestroy(s) == 0
        del out, val, y, named                           # freed after the stream's end
        torch.cuda.synchronize()
        assert torch.empty_like(x).fill_(1).sum() == x.numel()
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_calls_on_a_stream_that_ends_before_its_tensors():
    import _children
    assert _children.run_child(_foreign_stream_child)["ok"]


def _named_in_a_capture_child(rep):
    """Streams named inside a capture: the capturing one, as an object and as a handle, and one forked from it."""
    import torch
    torch.zeros(1, device="cuda")
    n, K = 300, 80
    e = engine(K, Device=0)
    c = e.cache(n)
    x, at = torch.randn(n, K, 2, device="cuda"), torch.randperm(n, device="cuda")
    val, out, out2, y = (torch.zeros_like(x) for _ in range(4))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cur = torch.cuda.current_stream()
        c.write(x, slots=at, values=val, stream=cur)
        c.read(out, slots=at, stream=cur.cuda_stream)
        side.wait_stream(cur)
        c.read(out2, slots=at.clone(), stream=side)
        e.dropout(x, 0.5, 3, out=y, stream=side.cuda_stream)
        cur.wait_stream(side)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (val, out, out2, y)]
        c.write(x, slots=at, values=val)                 # the program's own eager work
        e.dropout(x, 0.5, 3, out=y)
        torch.cuda.synchronize()
        assert all(torch.equal(a, val) for a in got[:3]) and torch.equal(got[3], y), i
    c.close()
    e.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_streams_named_inside_a_capture():
    import _children
    assert _children.run_child(_named_in_a_capture_child)["ok"]


# ------------------------------------------------------------------------------------------------ host memory in several pieces
def test_host_frames_of_several_staging_pieces(dev):  # noqa: F811
    """90 MB of host frames go through 32 MB of staging: bit for bit the device path, by slots (one named again in a later piece, padding) and
    in order, dense and apart, with dropout's counter running on."""
    K, n = 192, 30000
    e = engine(K)
    x = frames(n, K, 4)
    rng = np.random.default_rng(2)
    slots = rng.permutation(n + 100)[:n].astype(np.int64)
    slots[100], slots[n - 50] = slots[n - 7], slots[40]  # first and third piece
    slots[[5, 15000, n - 1]] = -1
    src, at = dev.up(x, "float64"), dev.up(slots, "int64")
    val, out, drop = (dev.up(np.full(x.shape, 9.0), "float64") for _ in range(3))
    c, h = e.cache(n + 100, 8, 16), e.cache(n + 100, 8, 16)
    c.write(src, slots=at, values=val)
    c.read(out, slots=at)
    c.read(drop, slots=at, p=0.3, seed=8, offset=1)
    want, want_val, want_drop = (dev.down(d, x.shape) for d in (out, val, drop))
    wide = np.full((n, K + 3, 2), 9.0)
    wide[:, 1:K + 1] = x
    values = np.full_like(x, 9.0)
    h.write(wide[:, 1:K + 1], slots=slots, values=values)
    assert np.array_equal(values, want_val)
    assert np.array_equal(h.read(np.full_like(x, 9.0), slots=slots), want)
    assert np.array_equal(h.read(np.full_like(x, 9.0), slots=slots, p=0.3, seed=8, offset=1), want_drop)
    wide[:] = 9.0
    h.read(wide[:, 1:K + 1], slots=at)                   # slots on the device
    assert np.array_equal(wide[:, 1:K + 1], want) and np.all(wide[:, 0] == 9) and np.all(wide[:, K + 1:] == 9)
    h.write(x, first=70)                                 # in order
    c.write(src, first=70)
    c.read(out, first=70)
    assert np.array_equal(h.read(np.empty_like(x), first=70), dev.down(out, x.shape))
    h.write(wide[:, 1:K + 1], slots=slots, values=wide[:, 1:K + 1])            # in place
    assert np.all(wide[:, 0] == 9) and np.all(wide[:, K + 1:] == 9) and np.all(wide[5, 1:K + 1] == 9)
    for k in (c, h):
        k.close()
    e.close()


@pytest.mark.parametrize("rows,cols,apart", [(9, 1_500_001, 3), (3, 5_000_003, 0), (2, 5_000_003, 4), (1, 9_000_001, 0)])
def test_host_dropout_of_several_staging_pieces(dev, rows, cols, apart):  # noqa: F811
    """Pieces of whole rows, and of one row where a row alone is more than the staging buffer."""
    e = engine(80)
    rng = np.random.default_rng(rows)
    wide = rng.normal(size=(rows, cols + apart))
    x = wide[:, apart:]
    src, out = dev.up(x, "float64"), dev.empty(x.size, "float64")
    e.dropout(src, 0.4, 77, 5, out=out)
    want = dev.down(out, x.shape)
    assert np.array_equal(want == 0, ref.dropped(0.4, 77, 5, x.size).reshape(x.shape))
    assert np.array_equal(e.dropout(x, 0.4, 77, 5), want)
    keep = wide[:, :apart].copy()
    e.dropout_backward(x, 0.4, 77, 5, out=x)
    assert np.array_equal(x, want) and np.array_equal(wide[:, :apart], keep)
    e.close()


def test_every_call_survives_a_launch_that_fails(dev):  # noqa: F811
    """Device and host memory, the second of several pieces, FromMel's upload and ToMel's write: status 8 each, and the next call works."""
    import gomel_amd
    from gomel_amd import _lib
    fail = _lib.lib().gomel_debug_fail_launch
    fail.restype, fail.argtypes = None, [ctypes.c_int]
    K, n = 192, 30000
    e = engine(K, GriffinLimIterations=2)
    c = e.cache(n)
    x = frames(n, K, 3)
    src, out = dev.up(x, "float64"), dev.empty(x.size, "float64")
    host, small, y = np.empty_like(x), np.empty((5, K, 2)), np.zeros(9_000_001)
    wave = np.random.default_rng(0).normal(size=30000)
    m = len(e.to_mel_batch([wave])[0]) // K
    b = gomel_amd.Batch(e, [40 * K])
    calls = {"write": (1, lambda: c.write(src)), "read": (1, lambda: c.read(out)), "read, dropout": (1, lambda: c.read(out, p=0.5)),
             "host write": (1, lambda: c.write(x[:5])), "second piece": (2, lambda: c.write(x)), "host read": (1, lambda: c.read(small)),
             "third piece": (3, lambda: c.read(host)), "dropout": (1, lambda: e.dropout(src, 0.5, 1, out=out)), "host dropout": (1, lambda: e.dropout(small, 0.5, 1)),
             "second piece of dropout": (2, lambda: e.dropout(y, 0.5, 1)), "backward": (1, lambda: e.dropout_backward(src, 0.5, 1, out=out)),
             "upload_cache": (1, lambda: b.upload_cache(c, np.arange(40))), "from_cache": (1, lambda: e.from_cache(c, [np.arange(40)])),
             "to_mel_cache": (1, lambda: e.to_mel_cache([wave], c, np.arange(m)))}
    for name, (nth, call) in calls.items():
        call()
        fail(nth)
        try:
            with pytest.raises(gomel_amd.GomelError) as err:
                call()
            assert err.value.status == 8, name
        finally:
            fail(0)
        if name == "upload_cache":
            with pytest.raises(gomel_amd.GomelError):
                b.run()                                  # not uploaded any more
        call()
    c.write(src)
    c.read(out)
    assert np.array_equal(c.read(host), dev.down(out, x.shape))
    b.close()
    c.close()
    e.close()


def _gate_child(rep):
    """Calls that wait for the caller's stream wait outside the gate: a persistent launch of another engine is let in meanwhile."""
    import threading
    import time
    import torch
    import gomel_amd
    torch.zeros(1, device="cuda")
    K = 80
    one = engine(K, Device=0, Resolut=1024, Window=256, MelFmax=8000, GriffinLimIterations=50)
    one.set_path(3)                                      # persistent
    one.set_precision(32)
    run = gomel_amd.Batch(one, [4 * K])
    run.upload([frames(4, K, 3).reshape(-1, 2)], None, [1])
    other = engine(K, Device=0)
    c = other.cache(64)
    c.write(frames(64, K, 1))
    b = gomel_amd.Batch(other, [40 * K])
    wave = np.random.default_rng(0).normal(size=30000)
    n = len(other.to_mel_batch([wave])[0]) // K
    side = torch.cuda.Stream()
    assert run.run_timed()["fast_path"] == 2
    for what in (lambda: b.upload_cache(c, np.arange(40), stream=side), lambda: other.to_mel_cache([wave], c, np.arange(n), stream=side)):
        what()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):                    # busy for a while, and the GPU is not
            for _ in range(20):
                torch.cuda._sleep(10_000_000)
        waiting = threading.Thread(target=what)
        t0 = time.perf_counter()
        waiting.start()
        time.sleep(0.005)
        paths = []
        while waiting.is_alive() and not side.query() and time.perf_counter() - t0 < 5:
            paths.append(run.run_timed()["fast_path"])
        waiting.join()
        assert len(paths) > 1 and 2 in paths, paths
        torch.cuda.synchronize()
    for k in (b, run, c, one, other):
        k.close()
    rep.result({"ok": True})


@pytest.mark.torch_child
@pytest.mark.guard(700)
def test_waiting_for_the_callers_stream_keeps_no_persistent_launch_out():
    import _children
    assert _children.run_child(_gate_child)["ok"]
