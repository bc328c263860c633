"""The spectrogram cache and dropout over the C ABI (gomel_cache_*, gomel_dropout* in include/gomel_hip.h: formulas and contract there).

What the calls take: numpy arrays (float64, float32, float16; copied through a staging buffer, the call returns when it is done), torch
tensors on the engine's device (those types and bfloat16; the call only queues kernels) and `DevicePointer`s.  A call runs on `stream`,
else on torch's current stream where torch is in use, else on the default stream.  There is no CPU fallback."""
import ctypes
import sys
from operator import index as _index     # any integer's value: Python's, numpy's, a torch scalar's

import numpy as np

from . import _lib
from ._lib import GomelError, check
from .mel import Batch, DevicePointer

_ON_DEVICE = 0x100           # GOMEL_DEVICE_MEMORY: nothing of the call is in host memory
_U64 = 0xFFFFFFFFFFFFFFFF
_FAR = 2 ** 63               # stands for every number of slots from there on: the library refuses it
_TYPES = {"float64": 0, "float32": 1, "float16": 2, "bfloat16": 3}
_torch = _forward_ad = None  # the modules torch and torch.autograd.forward_ad, once a tensor has been seen
_increment_version = None    # torch.autograd.graph.increment_version of an iterable of tensors
_Tensor = None               # its Tensor type
_torch_types, _int64 = {}, None
_raw_stream = None           # device index -> hipStream_t of torch's current stream


class _AnyLevel:
    """torch.autograd.forward_ad, where it does not say whether a level of dual tensors is open: every tensor is asked."""
    _current_level = 0

    @staticmethod
    def unpack_dual(t):
        return _torch.autograd.forward_ad.unpack_dual(t)


def _version_counter(torch):
    """torch.autograd.graph.increment_version without its wrapper (0.2 us), where that does the same."""
    try:
        with torch.inference_mode(False):        # (its tensors have no version)
            probe = torch.empty(0, device="cpu")
            torch._C._increment_version((probe,))
            if probe._version == 1:
                return torch._C._increment_version
    except (AttributeError, TypeError, RuntimeError):
        pass
    return torch.autograd.graph.increment_version


def _is_tensor(a):
    """Whether `a` is a torch tensor (torch is never imported for the question)."""
    global _torch, _Tensor, _int64, _raw_stream, _forward_ad, _increment_version
    if _Tensor is not None:
        return isinstance(a, _Tensor)
    if "torch" not in sys.modules or not hasattr(a, "data_ptr") or isinstance(a, DevicePointer):
        return False
    import torch
    _torch_types.update({torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3})
    _int64 = torch.int64
    _forward_ad = torch.autograd.forward_ad if hasattr(torch.autograd.forward_ad, "_current_level") else _AnyLevel
    _increment_version = _version_counter(torch)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    _torch, _Tensor = torch, torch.Tensor
    return isinstance(a, _Tensor)


def _torch_cuda():
    """torch.cuda where this process uses it, else None (torch may not be there, or be on its way in)."""
    cuda = getattr(sys.modules.get("torch"), "cuda", None)
    return cuda if cuda is not None and getattr(cuda, "is_initialized", bool)() else None


def _capturing(stream, device):
    """Whether torch's current stream, or the stream a call names, is being captured into a graph."""
    cuda = _torch_cuda()
    if cuda is None:
        return False
    with cuda.stream(cuda.current_stream(device) if stream is None else _as_stream(stream, device)):
        return cuda.is_current_stream_capturing()


def _stream(stream, device, engine_device):
    """The hipStream_t a call runs on: `stream` (an integer handle, or an object with .cuda_stream), else torch's current stream of the
    tensors' device -- of the engine's, where the call has no tensor: it follows the tensor calls before it --, else the default stream."""
    if stream is not None:
        return int(getattr(stream, "cuda_stream", stream))
    if device is not None:
        return _raw_stream(device)
    cuda = _torch_cuda()
    return 0 if cuda is None or engine_device < 0 else cuda.current_stream(engine_device).cuda_stream


def _as_stream(stream, device):
    """torch's stream object for a `stream` argument (an integer handle, or an object with .cuda_stream)."""
    cuda = sys.modules["torch"].cuda
    if isinstance(stream, cuda.Stream):
        return stream
    handle = int(getattr(stream, "cuda_stream", stream))
    return cuda.ExternalStream(handle, device=device) if handle else cuda.default_stream(device)


def _used_on(stream, *arrays):
    """Keeps the memory of these tensors, should they be dropped now, from being handed on before a call on a named stream is through with
    it.  On a stream of torch's its allocator is told.  It would ask a foreign one (an integer handle) when the tensors are freed, which
    may be after the stream's end: there torch's current stream waits for the call."""
    tensors = [a for a in arrays if isinstance(a, _Tensor)] if _Tensor is not None else ()
    if not tensors:
        return
    cuda, device = _torch.cuda, tensors[0].get_device()
    if isinstance(stream, cuda.Stream) and not isinstance(stream, cuda.ExternalStream):
        for a in tensors:
            a.record_stream(stream)
    elif int(getattr(stream, "cuda_stream", stream)) != _raw_stream(device) and not _capturing(None, device) and not _capturing(stream, device):
        cuda.current_stream(device).wait_stream(_as_stream(stream, device))


def _device_of(engine_device, *devices):
    """The device of a call's tensors (None: there are none); they have to be on one device, the engine's."""
    got = None
    for d in devices:
        if d is not None:
            if (got is not None and d != got) or (engine_device >= 0 and d != engine_device):
                raise ValueError("a tensor on device %d was handed to a call on device %d" % (d, engine_device if engine_device >= 0 else got))
            got = d
    return got


def _rows(a, cols, what, write=False):
    """(address, type code, row stride in elements, rows, device) of an array of rows of `cols` elements.  Rows may be apart; the
    elements of a row are consecutive.  device: a torch tensor's, None otherwise."""
    device = None
    if _is_tensor(a) if _Tensor is None else isinstance(a, _Tensor):
        device, t = a.get_device(), _torch_types.get(a.dtype)
        if device < 0:
            raise ValueError("%s: a torch tensor must be on the GPU (numpy arrays are taken from host memory)" % what)
        if t is not None and a.is_contiguous():
            rows, rest = divmod(a.numel(), cols)
            if not rest:
                return a.data_ptr(), t, cols, rows, device
        strides, ptr = a.stride(), a.data_ptr()
    elif isinstance(a, DevicePointer):
        t, n = _TYPES.get(a.dtype), a.numel()
        if t is None or n % cols:
            raise ValueError("%s: a DevicePointer of float64 / float32 / float16 / bfloat16 with whole rows of %d elements is needed" % (what, cols))
        return a.data_ptr(), t, cols, n // cols, None
    elif isinstance(a, np.ndarray):
        t, strides, ptr = _TYPES.get(a.dtype.name), [s // a.itemsize for s in a.strides], a.ctypes.data
        if any(s % a.itemsize for s in a.strides) or not a.dtype.isnative:
            t = None
        if write and not a.flags.writeable:
            raise ValueError("%s: the array is read-only" % what)
    elif hasattr(a, "data_ptr"):
        raise ValueError("%s: a torch tensor must be on the GPU (numpy arrays are taken from host memory)" % what)
    else:
        raise TypeError("%s: a numpy array, a torch CUDA tensor or a DevicePointer is needed, not %s" % (what, type(a).__name__))
    if t is None:
        raise ValueError("%s: float64, float32, float16 or bfloat16 is needed, not %s" % (what, a.dtype))
    shape = tuple(a.shape)
    n = 1
    for s in shape:
        n *= s
    if n % cols:
        raise ValueError("%s: whole rows of %d elements are needed, not shape %s" % (what, cols, shape))
    rows = n // cols
    if rows == 0:
        return ptr, t, cols, 0, device
    # innermost dimensions that make up one row have to be dense; what remains has to step evenly from row to row
    inner, i = 1, len(shape)
    while inner < cols:
        i -= 1
        if shape[i] != 1 and strides[i] != inner:
            raise ValueError("%s: the elements of a row must be consecutive" % what)
        inner *= shape[i]
        if inner > cols:                     # [n * NumMels, 2]: a dense block of several rows
            if inner % cols:
                raise ValueError("%s: whole rows of %d elements are needed, not shape %s" % (what, cols, shape))
            if inner != n:
                raise ValueError("%s: rows of %d elements cannot be stepped through evenly" % (what, cols))
            return ptr, t, cols, rows, device
    step, count = None, 1
    for k in range(i - 1, -1, -1):
        if shape[k] == 1:
            continue
        if step is None:
            step, count = strides[k], shape[k]
        elif strides[k] == step * count:
            count *= shape[k]
        else:
            raise ValueError("%s: rows of %d elements cannot be stepped through evenly" % (what, cols))
    if step is None:
        step = cols
    if step < cols:
        raise ValueError("%s: rows overlap" % what)
    return ptr, t, step, rows, device


def _output(a, what):
    """Refuses an output that autograd keeps track of: it does not see what a call writes."""
    if _wants_grad(a):
        raise ValueError("%s: a tensor that requires a gradient or carries a tangent cannot be written to" % what)


def _written(a):
    """Tells autograd that a call has written to `a`: where it holds the tensor's old values for a backward pass, that pass now raises."""
    if _Tensor is not None and isinstance(a, _Tensor):
        _increment_version((a,))


def _host_slots(slots, what):
    a = np.asarray(slots)
    if a.dtype.kind not in "iu" and a.size:
        raise ValueError("%s: integers are needed, not %s" % (what, a.dtype))
    if a.dtype.kind == "u" and a.size and int(a.max()) > 2 ** 63 - 1:
        raise ValueError("%s: beyond int64" % what)
    return np.ascontiguousarray(a, dtype=np.int64).reshape(-1)


def _slots(slots, n, what="slots"):
    """(address, the array that has to stay alive, device) of one int64 per frame."""
    if _is_tensor(slots) if _Tensor is None else isinstance(slots, _Tensor):
        device = slots.get_device()
        if device < 0 or slots.dtype != _int64 or not slots.is_contiguous() or slots.numel() != n:
            raise ValueError("%s: a contiguous int64 CUDA tensor with %d elements is needed" % (what, n))
        return slots.data_ptr(), slots, device
    if isinstance(slots, DevicePointer):
        if slots.dtype != "int64" or slots.numel() != n:
            raise ValueError("%s: a DevicePointer of %d int64 is needed" % (what, n))
        return slots.data_ptr(), slots, None
    a = _host_slots(slots, what)
    if a.size != n:
        raise ValueError("%s: one slot per frame is needed (%d frames, %d slots)" % (what, n, a.size))
    return (a.ctypes.data if n else 0), a, None


def _far(first):
    if first < 0:
        raise ValueError("first is negative")
    return _FAR


_left = []                   # (cache, device) of those closed or collected while torch's current stream was being captured


def _destroy_left(device):
    if _left and not _capturing(None, device):
        for k in [k for k in _left if not _capturing(None, k[1])]:
            try:
                _left.remove(k)
            except ValueError:               # another thread has it
                continue
            _lib.lib().gomel_cache_destroy(k[0])


class Cache:
    """gomel_cache: `n_slots` slots of one quantised frame ([NumMels][2] values) in the device's memory.  `bits` 8 or 4 per value; `group`
    bands share a minimum and a step (0 = the whole frame, or 8, 16, 32, 64).  Pages and their tables are the caller's: `slots` names one
    slot per frame (negative: padding, the frame is left alone), or frames go to the slots first, first + 1, ..."""

    def __init__(self, engine, n_slots, bits=8, group=0):
        self._c = ctypes.c_void_p()
        self.n_slots, self.bits, self.group, self.num_mels = int(n_slots), int(bits), int(group), int(engine.cfg.num_mels)
        self.device = int(engine.cfg.device)
        if self.n_slots < 0:
            raise ValueError("n_slots is negative")
        if _capturing(None, self.device):        # as the library's calls that wait: it would end the capture
            raise GomelError(1, "gomel_cache_create")
        _destroy_left(self.device)
        L = _lib.lib()
        held = min(self.n_slots, _FAR), *(v if abs(v) < 2 ** 31 else -1 for v in (self.bits, self.group))    # (ctypes would cut the rest off)
        self.frame_bytes = L.gomel_cache_frame_bytes(ctypes.byref(engine.cfg), *held[1:])
        check(L.gomel_cache_create(engine._h, *held, ctypes.byref(self._c)), "gomel_cache_create")
        self._write, self._read = L.gomel_cache_write, L.gomel_cache_read

    def write(self, frames, slots=None, first=0, values=None, stream=None):
        """Quantises `frames` ([n, NumMels, 2] or [n * NumMels, 2]) into their slots.  `values` (same shape and type; may be `frames` itself)
        receives what the cache now stands for, and is returned.  No gradient goes through the quantiser: frames that require one are refused
        where `values` is given (write frames.detach(); straight through, frames + (values - frames).detach())."""
        cols = 2 * self.num_mels
        ptr, t, stride, n, dev = _rows(frames, cols, "frames")
        sp, keep, sdev = (0, None, None) if slots is None else _slots(slots, n)
        vp, vs, vdev = 0, cols, None
        if values is not None:
            if _wants_grad(frames):
                raise ValueError("values: not with frames that require a gradient or carry a tangent")
            _output(values, "values")
            vp, vt, vs, vn, vdev = _rows(values, cols, "values", write=True)
            if vt != t or vn != n:
                raise ValueError("values: the frames' type and number of frames are needed")
        if not 0 <= first < _FAR:
            first = _far(first)
        on = self.device
        if dev == on and (values is None or vdev == on) and (slots is None or sdev == on):
            t |= _ON_DEVICE
        else:
            on = _device_of(on, dev, vdev, sdev)
        if _left:
            _destroy_left(self.device)
        rc = self._write(self._c, t, ptr, stride, n, sp, first, vp, vs, _stream(stream, on, self.device))
        _written(values)
        if stream is not None:
            _used_on(stream, frames, values, slots)
        if rc:
            check(rc, "gomel_cache_write")
        return values

    def read(self, out, slots=None, first=0, p=0.0, seed=0, offset=0, stream=None):
        """Dequantises frames into `out` ([n, NumMels, 2] or [n * NumMels, 2]) and returns it.  p > 0: with dropout, as Engine.dropout of
        the dense result."""
        _output(out, "out")
        ptr, t, stride, n, dev = _rows(out, 2 * self.num_mels, "out", write=True)
        sp, keep, sdev = (0, None, None) if slots is None else _slots(slots, n)
        if not 0 <= first < _FAR:
            first = _far(first)
        on = self.device
        if dev == on and (slots is None or sdev == on):
            t |= _ON_DEVICE
        else:
            on = _device_of(on, dev, sdev)
        if _left:
            _destroy_left(self.device)
        rc = self._read(self._c, t, ptr, stride, n, sp, first, p, _index(seed) & _U64, _index(offset) & _U64, _stream(stream, on, self.device))
        _written(out)
        if stream is not None:
            _used_on(stream, out, slots)
        if rc:
            check(rc, "gomel_cache_read")
        return out

    def bad_slots(self):
        """Frames skipped since the last call because a slot in device memory was not one of the cache's (gomel_cache_bad_slots)."""
        if self._c and _capturing(None, self.device):
            raise GomelError(1, "bad_slots")
        n = ctypes.c_uint64(0)
        check(_lib.lib().gomel_cache_bad_slots(self._c, ctypes.byref(n)), "gomel_cache_bad_slots")
        return n.value

    def close(self):
        """Gives the memory back -- in a capture (gomel_cache_destroy waits for the device, which would end it) when the next call of any
        cache is made outside one."""
        if self._c:
            later = _capturing(None, self.device)
            c, self._c = self._c, ctypes.c_void_p()
            if later:
                _left.append((c, self.device))
            else:
                _destroy_left(self.device)
                check(_lib.lib().gomel_cache_destroy(c), "gomel_cache_destroy")

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------------------------------------ FromMel / ToMel and the cache
def batch_upload_cache(batch, cache, slots, x0s=None, seeds=None, stream=None):
    sp, keep, dev = _slots(slots, sum(batch.n_pairs) // batch.engine.cfg.num_mels)
    xp, xs, seed_p = batch._x0_args(x0s, seeds)
    check(_lib.lib().gomel_batch_upload_cache(batch._b, cache._c, sp, xp, seed_p, _stream(stream, _device_of(cache.device, dev), cache.device)),
          "gomel_batch_upload_cache")
    del xs, keep


def _joined(slots, stream, engine_device):
    """(all utterances' slots as one array, how many each has)"""
    tensors = sum(_is_tensor(s) for s in slots)
    if not tensors and len(slots) == 1 and isinstance(slots[0], DevicePointer):
        return slots[0], [slots[0].numel()]
    if not tensors and not any(isinstance(s, DevicePointer) for s in slots):
        arrays = [_host_slots(s, "slots") for s in slots]
        return np.concatenate(arrays), [a.size for a in arrays]
    if tensors != len(slots):                    # (DevicePointers of several utterances: Batch.upload_cache takes them as one)
        raise ValueError("slots: of several utterances, either all in host memory or all as int64 CUDA tensors")
    if any(s.dtype != _int64 or not s.is_cuda for s in slots):
        raise ValueError("slots: int64 CUDA tensors are needed (numpy arrays are taken from host memory)")
    on = _device_of(engine_device, *[s.get_device() for s in slots])
    # in the order of the call's stream: there the slots are ready, and there they are read
    with _torch.cuda.stream(_torch.cuda.current_stream(on) if stream is None else _as_stream(stream, on)):
        return _torch.cat([s.reshape(-1) for s in slots]), [s.numel() for s in slots]


def from_cache(engine, cache, slots, x0s=None, seeds=None, stream=None):
    slots = list(slots)
    if not slots:
        return []
    if _capturing(stream, cache.device):         # as gomel_batch_upload_cache, before a batch is allocated
        raise GomelError(1, "from_cache")
    flat, counts = _joined(slots, stream, cache.device)
    b = Batch(engine, [c * engine.cfg.num_mels for c in counts])
    try:
        b.upload_cache(cache, flat, x0s, seeds, stream)
        b.run()
        return b.download()
    finally:
        b.close()


def to_mel_cache(engine, waves, cache, slots, stream=None):
    L = _lib.lib()
    ws = [np.ascontiguousarray(w, dtype=np.float64) for w in waves]
    counts = [L.gomel_to_mel_pairs(ctypes.byref(engine.cfg), w.size) // engine.cfg.num_mels for w in ws]
    total = sum(counts)
    sp, keep, dev = _slots(slots, total)
    wp = (_lib.c_double_p * len(ws))(*[w.ctypes.data_as(_lib.c_double_p) for w in ws])
    ns = (ctypes.c_size_t * len(ws))(*[w.size for w in ws])
    check(L.gomel_to_mel_cache(engine._h, len(ws), wp, ns, cache._c, sp, total, _stream(stream, _device_of(cache.device, dev), cache.device)),
          "gomel_to_mel_cache")
    del keep
    return counts


# ------------------------------------------------------------------------------------------------ dropout
def _flat(a, what, write=False):
    """(address, type code, row stride, rows, cols, device) of any array that is dense, or whose rows (its last dimension) are."""
    if _is_tensor(a):
        n, dense = a.numel(), a.is_contiguous()
    elif isinstance(a, np.ndarray):
        n, dense = a.size, a.flags.c_contiguous
    else:
        n, dense = (a.numel() if isinstance(a, DevicePointer) else 1), True
    if dense or n == 0:
        ptr, t, _, _, device = _rows(a, n or 1, what, write)
        return ptr, t, n, 1, n, device
    cols = int(a.shape[-1])
    ptr, t, stride, rows, device = _rows(a, cols, what, write)
    return ptr, t, stride, rows, cols, device


def _dropout(fn, where, engine, x, p, seed, offset, out, stream):
    device = engine.cfg.device
    if out is not None and (_Tensor is None or not isinstance(out, _Tensor) or out.requires_grad or _forward_ad._current_level >= 0):
        _output(out, "out")
    if out is not None and _Tensor is not None and isinstance(x, _Tensor) and isinstance(out, _Tensor) and x.is_contiguous() and out.is_contiguous() and x.shape == out.shape and x.dtype == out.dtype:
        t, n = _torch_types.get(x.dtype), x.numel()                       # two dense tensors: nothing to work out
        if t is not None and n and device == x.get_device() == out.get_device():
            rc = fn(engine._h, t | _ON_DEVICE, x.data_ptr(), n, out.data_ptr(), n, 1, n, p, _index(seed) & _U64, _index(offset) & _U64,
                    _raw_stream(device) if stream is None else _stream(stream, device, device))
            _increment_version((out,))
            if stream is not None:
                _used_on(stream, x, out)
            if rc:
                check(rc, where)
            return out
    ptr, t, xs, rows, cols, dev = _flat(x, "x")
    if out is None:
        if isinstance(x, DevicePointer):
            raise ValueError("out: a DevicePointer needs one")
        if stream is not None and dev is not None:       # torch would hand the new tensor's memory on in the order of its own stream
            raise ValueError("out: needed where a stream is named")
        out = np.empty(x.shape, x.dtype) if dev is None else _torch.empty(x.shape, dtype=x.dtype, device=x.device)
    optr, ot, os_, orows, ocols, odev = _flat(out, "out", write=True)
    if ot != t or getattr(out, "shape", None) != getattr(x, "shape", None) or rows * cols != orows * ocols:
        raise ValueError("out: x's type and shape are needed")
    if rows != orows:                        # one of the two is dense: walk it by the other's rows
        if rows == 1:
            rows, cols, xs = orows, ocols, ocols
        else:
            os_ = cols
    on = _device_of(device, dev, odev)
    if on == device and dev is not None and odev is not None:
        t |= _ON_DEVICE
    rc = fn(engine._h, t, ptr, xs, optr, os_, rows, cols, p, _index(seed) & _U64, _index(offset) & _U64, _stream(stream, on, device))
    _written(out)
    if stream is not None:
        _used_on(stream, x, out)
    if rc:
        check(rc, where)
    return out


_function = None


def _dropout_function():
    """torch.autograd.Function over the two calls, made when the first gradient is asked for (torch is optional)."""
    global _function
    if _function is None:
        import torch

        class Dropout(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, engine, p, seed, offset, back):
                ctx.args, ctx.back = (engine, p, seed, offset), back
                fn = _lib.lib().gomel_dropout_backward if back else _lib.lib().gomel_dropout
                return _dropout(fn, "gomel_dropout_backward" if back else "gomel_dropout", engine, x, p, seed, offset, None, None)

            @staticmethod
            def backward(ctx, dy):
                return (Dropout.apply(dy.contiguous(), *ctx.args, not ctx.back),) + (None,) * 5

            @staticmethod
            def jvp(ctx, dx, *rest):                     # linear in x: the tangent goes the same way
                return Dropout.apply(dx.contiguous(), *ctx.args, ctx.back)

        _function = Dropout
    return _function


def _wants_grad(x):
    """Whether autograd has to see what is computed from x: in reverse mode, or in forward mode (x carries a tangent)."""
    if not (_is_tensor(x) if _Tensor is None else isinstance(x, _Tensor)):
        return False
    if x.requires_grad and _torch.is_grad_enabled():
        return True
    return _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(x).tangent is not None


def dropout(engine, x, p, seed, offset=0, out=None, stream=None):
    if _wants_grad(x):
        if out is not None or stream is not None:
            raise ValueError("out, stream: not with a tensor that requires a gradient or carries a tangent")
        return _dropout_function().apply(x, engine, p, seed, offset, False)
    return _dropout(_lib.lib().gomel_dropout, "gomel_dropout", engine, x, p, seed, offset, out, stream)


def dropout_backward(engine, dy, p, seed, offset=0, out=None, stream=None):
    if _wants_grad(dy):
        if out is not None or stream is not None:
            raise ValueError("out, stream: not with a tensor that requires a gradient or carries a tangent")
        return _dropout_function().apply(dy, engine, p, seed, offset, True)
    return _dropout(_lib.lib().gomel_dropout_backward, "gomel_dropout_backward", engine, dy, p, seed, offset, out, stream)
