"""The spectrogram cache and dropout over the C ABI (gomel_cache_*, gomel_dropout* in include/gomel_hip.h: formulas and contract there).

What the calls take: numpy arrays (float64, float32, float16; copied through a staging buffer, the call returns when it is done), torch
tensors on the engine's device (those types and bfloat16; the call queues kernels on torch's current stream, or on `stream`) and
`DevicePointer`s.  There is no CPU fallback."""
import ctypes
import sys

import numpy as np

from . import _lib
from ._lib import check
from .mel import Batch, DevicePointer, _is_device_tensor

_TYPES = {"float64": 0, "float32": 1, "float16": 2, "bfloat16": 3}
_torch_types = {}


def _torch_type(dtype):
    """The element type's code of a torch dtype, None for one the library does not take."""
    if not _torch_types:
        import torch
        _torch_types.update({torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3})
    return _torch_types.get(dtype)


def _stream(stream, *arrays):
    """The hipStream_t a call runs on: `stream` (an integer handle, or an object with .cuda_stream), else torch's current stream of the
    first torch tensor's device, else the default stream."""
    if stream is not None:
        return int(getattr(stream, "cuda_stream", stream))
    for a in arrays:
        if a is not None and not isinstance(a, (np.ndarray, DevicePointer)):
            import torch
            return torch.cuda.current_stream(a.device).cuda_stream
    return 0


def _rows(a, cols, what, write=False):
    """(address, type code, row stride in elements, rows) of an array of rows of `cols` elements.  Rows may be apart; the elements of
    a row are consecutive."""
    if isinstance(a, DevicePointer):
        t, n = _TYPES.get(a.dtype), a.numel()
        if t is None or n % cols:
            raise ValueError("%s: a DevicePointer of float64 / float32 / float16 / bfloat16 with whole rows of %d elements is needed" % (what, cols))
        return a.data_ptr(), t, cols, n // cols
    if isinstance(a, np.ndarray):
        t, strides, ptr = _TYPES.get(a.dtype.name), [s // a.itemsize for s in a.strides], a.ctypes.data
        if any(s % a.itemsize for s in a.strides) or not a.dtype.isnative:
            t = None
        if write and not a.flags.writeable:
            raise ValueError("%s: the array is read-only" % what)
    elif hasattr(a, "data_ptr"):
        if not a.is_cuda:
            raise ValueError("%s: a torch tensor must be on the GPU (numpy arrays are taken from host memory)" % what)
        t, strides, ptr = _torch_type(a.dtype), a.stride(), a.data_ptr()
    else:
        raise TypeError("%s: a numpy array, a torch CUDA tensor or a DevicePointer is needed, not %s" % (what, type(a).__name__))
    if t is None:
        raise ValueError("%s: float64, float32, float16 or bfloat16 is needed, not %s" % (what, a.dtype))
    shape = tuple(a.shape)
    n = 1
    for s in shape:
        n *= s
    if n % cols or n == 0 and cols == 0:
        raise ValueError("%s: whole rows of %d elements are needed, not shape %s" % (what, cols, shape))
    rows = n // cols
    if rows == 0:
        return ptr, t, cols, 0
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
            return ptr, t, cols, rows
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
    return ptr, t, step, rows


def _slots(slots, n, what="slots"):
    """(address, the array that has to stay alive) of one int64 per frame."""
    if isinstance(slots, DevicePointer):
        if slots.dtype != "int64" or slots.numel() != n:
            raise ValueError("%s: a DevicePointer of %d int64 is needed" % (what, n))
        return slots.data_ptr(), slots
    if hasattr(slots, "data_ptr"):
        if not slots.is_cuda or str(slots.dtype) != "torch.int64" or not slots.is_contiguous() or slots.numel() != n:
            raise ValueError("%s: a contiguous int64 CUDA tensor with %d elements is needed" % (what, n))
        return slots.data_ptr(), slots
    a = np.asarray(slots)
    if a.dtype.kind not in "iu" and a.size:
        raise ValueError("%s: integers are needed, not %s" % (what, a.dtype))
    a = np.ascontiguousarray(a, dtype=np.int64).reshape(-1)
    if a.size != n:
        raise ValueError("%s: one slot per frame is needed (%d frames, %d slots)" % (what, n, a.size))
    return (a.ctypes.data if n else 0), a


def _same_device(engine_device, *arrays):
    for a in arrays:
        if a is not None and not isinstance(a, (np.ndarray, DevicePointer)) and hasattr(a, "device") and engine_device >= 0:
            if a.device.index != engine_device:
                raise ValueError("a tensor on %s was handed to an engine on device %d" % (a.device, engine_device))


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
        L = _lib.lib()
        self.frame_bytes = L.gomel_cache_frame_bytes(ctypes.byref(engine.cfg), self.bits, self.group)
        check(L.gomel_cache_create(engine._h, self.n_slots, self.bits, self.group, ctypes.byref(self._c)), "gomel_cache_create")
        self._write, self._read = L.gomel_cache_write, L.gomel_cache_read

    def write(self, frames, slots=None, first=0, values=None, stream=None):
        """Quantises `frames` ([n, NumMels, 2] or [n * NumMels, 2]) into their slots.  `values` (same shape and type; may be `frames` itself)
        receives what the cache now stands for, and is returned."""
        cols = 2 * self.num_mels
        ptr, t, stride, n = _rows(frames, cols, "frames")
        sp, keep = (0, None) if slots is None else _slots(slots, n)
        vp, vs = 0, cols
        if values is not None:
            vp, vt, vs, vn = _rows(values, cols, "values", write=True)
            if vt != t or vn != n:
                raise ValueError("values: the frames' type and number of frames are needed")
        if first < 0:
            raise ValueError("first is negative")
        _same_device(self.device, frames, values, slots)
        rc = self._write(self._c, t, ptr, stride, n, sp, first, vp, vs, _stream(stream, frames, values, keep))
        if rc:
            check(rc, "gomel_cache_write")
        return values

    def read(self, out, slots=None, first=0, p=0.0, seed=0, offset=0, stream=None):
        """Dequantises frames into `out` ([n, NumMels, 2] or [n * NumMels, 2]) and returns it.  p > 0: with dropout, as Engine.dropout of
        the dense result."""
        ptr, t, stride, n = _rows(out, 2 * self.num_mels, "out", write=True)
        sp, keep = (0, None) if slots is None else _slots(slots, n)
        if first < 0:
            raise ValueError("first is negative")
        _same_device(self.device, out, slots)
        rc = self._read(self._c, t, ptr, stride, n, sp, first, p, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, _stream(stream, out, keep))
        if rc:
            check(rc, "gomel_cache_read")
        return out

    def bad_slots(self):
        """Frames skipped so far because a slot in device memory was not one of the cache's (gomel_cache_bad_slots)."""
        n = ctypes.c_uint64(0)
        check(_lib.lib().gomel_cache_bad_slots(self._c, ctypes.byref(n)), "gomel_cache_bad_slots")
        return n.value

    def close(self):
        if self._c:
            c, self._c = self._c, ctypes.c_void_p()
            check(_lib.lib().gomel_cache_destroy(c), "gomel_cache_destroy")

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------------------------------------ FromMel / ToMel and the cache
def batch_upload_cache(batch, cache, slots, x0s=None, seeds=None, stream=None):
    sp, keep = _slots(slots, sum(batch.n_pairs) // batch.engine.cfg.num_mels)
    xp, xs, seed_p = batch._x0_args(x0s, seeds)
    check(_lib.lib().gomel_batch_upload_cache(batch._b, cache._c, sp, xp, seed_p, _stream(stream, keep)), "gomel_batch_upload_cache")
    del xs


def from_cache(engine, cache, slots, x0s=None, seeds=None, stream=None):
    counts = [int(s.numel()) if hasattr(s, "numel") else len(s) for s in slots]
    if not counts:
        return []
    if any(_is_device_tensor(s) for s in slots):
        import torch
        flat = torch.cat([s.reshape(-1) for s in slots])
    else:
        flat = np.concatenate([np.asarray(s, dtype=np.int64).reshape(-1) for s in slots])
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
    sp, keep = _slots(slots, total)
    wp = (_lib.c_double_p * len(ws))(*[w.ctypes.data_as(_lib.c_double_p) for w in ws])
    ns = (ctypes.c_size_t * len(ws))(*[w.size for w in ws])
    check(L.gomel_to_mel_cache(engine._h, len(ws), wp, ns, cache._c, sp, total, _stream(stream, keep)), "gomel_to_mel_cache")
    return counts


# ------------------------------------------------------------------------------------------------ dropout
def _flat(a, what, write=False):
    """(address, type code, row stride, rows, cols) of any array that is dense, or whose rows (its last dimension) are."""
    if isinstance(a, DevicePointer):
        ptr, t, _, _ = _rows(a, 1, what, write)
        return ptr, t, a.numel(), 1, a.numel()
    n = 1
    for s in a.shape:
        n *= s
    dense = a.flags.c_contiguous if isinstance(a, np.ndarray) else (a.is_contiguous() if hasattr(a, "is_contiguous") else False)
    if dense or n == 0:
        ptr, t, _, _ = _rows(a, max(n, 1), what, write) if n else _rows(a, 1, what, write)
        return ptr, t, n, 1, n
    cols = int(a.shape[-1])
    ptr, t, stride, rows = _rows(a, cols, what, write)
    return ptr, t, stride, rows, cols


def _dropout(fn, where, engine, x, p, seed, offset, out, stream):
    ptr, t, xs, rows, cols = _flat(x, "x")
    if out is None:
        if isinstance(x, DevicePointer):
            raise ValueError("out: a DevicePointer needs one")
        if isinstance(x, np.ndarray):
            out = np.empty(x.shape, x.dtype)
        else:
            import torch
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    optr, ot, os_, orows, ocols = _flat(out, "out", write=True)
    if ot != t or getattr(out, "shape", None) != getattr(x, "shape", None) or rows * cols != orows * ocols:
        raise ValueError("out: x's type and shape are needed")
    if (rows, cols) != (orows, ocols):       # one of the two is dense: walk it by the other's rows
        if rows == 1:
            rows, cols, xs = orows, ocols, ocols
        else:
            os_ = cols
    _same_device(int(engine.cfg.device), x, out)
    rc = fn(engine._h, t, ptr, xs, optr, os_, rows, cols, p, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, _stream(stream, x, out))
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
            def forward(ctx, x, engine, p, seed, offset, stream, back):
                ctx.args = (engine, p, seed, offset, stream, not back)
                fn = _lib.lib().gomel_dropout_backward if back else _lib.lib().gomel_dropout
                return _dropout(fn, "gomel_dropout_backward" if back else "gomel_dropout", engine, x, p, seed, offset, None, stream)

            @staticmethod
            def backward(ctx, dy):
                engine, p, seed, offset, stream, back = ctx.args
                return Dropout.apply(dy if dy.is_contiguous() else dy.contiguous(), engine, p, seed, offset, stream, back), None, None, None, None, None, None

        _function = Dropout
    return _function


def _wants_grad(x):
    return "torch" in sys.modules and getattr(x, "requires_grad", False) and sys.modules["torch"].is_grad_enabled()


def dropout(engine, x, p, seed, offset=0, out=None, stream=None):
    if _wants_grad(x):
        if out is not None:
            raise ValueError("out: not with a tensor that requires a gradient")
        return _dropout_function().apply(x, engine, p, seed, offset, stream, False)
    return _dropout(_lib.lib().gomel_dropout, "gomel_dropout", engine, x, p, seed, offset, out, stream)


def dropout_backward(engine, dy, p, seed, offset=0, out=None, stream=None):
    if _wants_grad(dy):
        if out is not None:
            raise ValueError("out: not with a tensor that requires a gradient")
        return _dropout_function().apply(dy, engine, p, seed, offset, stream, True)
    return _dropout(_lib.lib().gomel_dropout_backward, "gomel_dropout_backward", engine, dy, p, seed, offset, out, stream)
