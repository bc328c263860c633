"""The spectrogram cache and dropout from their definitions, in numpy float64 / uint64: what the tests hold the kernels to.

Tolerances of a value read: lo + q * step is one fused multiply-add in fp32 (fp64 for float64), rounded once more to a 16-bit type;
dropout's factor is an fp32 number and its product is rounded: half a unit each, relative to the value -- 2^-24 per fp32 rounding, 2^-11
for float16, 2^-8 for bfloat16, 2^-53 for float64 -- plus half the smallest subnormal of the type."""
import numpy as np

GAMMA = 0x9E3779B97F4A7C15
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 5e-324, "float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def to_bf16(a):
    """float32 -> the bits of bfloat16 (nearest even; NaN stays NaN)."""
    b = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)
    r = ((b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (np.ascontiguousarray(u, dtype=np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def quantise(x, bits, group):
    """x [n][K][2] float64 -> (codes [n][K][2], lo, step [n][groups] float32)."""
    n, K, _ = x.shape
    g = group or K
    G, levels = -(-K // g), 2 ** bits - 1
    codes = np.zeros(x.shape, dtype=np.int64)
    lo, step = np.zeros((n, G), np.float32), np.zeros((n, G), np.float32)
    big = float(np.finfo(np.float32).max)
    with np.errstate(all="ignore"):
        for r in range(n):
            for j in range(G):
                v = x[r, j * g:(j + 1) * g]
                fin = v[np.isfinite(v)]
                if np.isnan(v).any() or (fin.size == 0 and np.isposinf(v).any() and np.isneginf(v).any()):
                    lo[r, j] = np.nan
                    continue
                if fin.size == 0:
                    lo[r, j] = np.inf if np.isposinf(v).any() else -np.inf
                    continue
                a = np.float32(np.clip(np.float64(np.float32(fin.min())), -big, big))
                b = np.float32(np.clip(np.float64(np.float32(fin.max())), -big, big))
                d = np.float32((np.float64(b) - np.float64(a)) / levels)
                lo[r, j], step[r, j] = a, d
                if d > 0:
                    q = np.rint((v - np.float64(a)) / np.float64(d))
                    codes[r, j * g:(j + 1) * g] = np.clip(q, 0, levels).astype(np.int64)
    return codes, lo, step


def stands_for(x, bits, group):
    """What frames x [n][K][2] (float64 values) read as, in float64."""
    K = x.shape[1]
    q, lo, step = quantise(x, bits, group)
    of = np.arange(K) // (group or K)
    with np.errstate(invalid="ignore"):
        return lo[:, of, None].astype(np.float64) + q * step[:, of, None].astype(np.float64)


def dropped(p, seed, offset, count):
    """Which of the elements offset ... offset + count - 1 (mod 2^64) are dropped."""
    e = np.uint64(offset & (2 ** 64 - 1)) + np.arange(count, dtype=np.uint64)
    with np.errstate(over="ignore"):
        z = np.uint64(seed & (2 ** 64 - 1)) + ((e >> np.uint64(1)) + np.uint64(1)) * np.uint64(GAMMA)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    u = np.where(e & np.uint64(1), z >> np.uint64(32), z & np.uint64(0xFFFFFFFF))
    return u < np.uint64(int(np.rint(p * 2.0 ** 32)))


def close(got, want, dtype, roundings):
    """got within `roundings` fp32 (fp64 for float64) roundings and one of dtype's; NaN and infinities in the same places.  `want` may be
    (want, bound): the operands' magnitude, which the reference's own sum in float64 loses to (two roundings of 2^-53 each)."""
    want, bound = want if isinstance(want, tuple) else (want, np.abs(want))
    got, half = np.asarray(got, dtype=np.float64), HALF[dtype] if dtype == "float64" else 2.0 ** -24
    top = {"float64": np.finfo(np.float64).max, "float32": float(np.finfo(np.float32).max), "float16": 65504.0, "bfloat16": 3.3895313892515355e38}[dtype]
    with np.errstate(invalid="ignore"):
        tol = np.abs(want) * (roundings * half * 1.001 + HALF[dtype] * 1.01) + bound * 2.0 ** -52 + 2 * TINY[dtype]
        same = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
        same |= np.isinf(got) & (np.abs(want) >= top) & (np.sign(got) == np.sign(want))      # a value beyond the type's range rounds to infinity
    return bool(same.all())
