"""Work and timing cases of the spectrogram cache (frames quantised as they are written, read back dequantised) and of dropout from a
counter-based generator.

A frame is [K][2] values, K = NumMels: the log-mel pairs that ToMel makes and FromMel takes.  L = 2**bits - 1.  Written, each group of
bands (both channels; `group` 0 = the whole frame, the last group may be short) keeps lo = min and step = fl32((max - lo) / L) in 32 bits
and q = rint((x - lo) / step) in `bits` bits, ties to even; read, a value is lo + q * step.  Dropout drops element e (dense index +
offset) iff the 32 bits that splitmix64 gives for it (seed + (e/2 + 1) * 0x9E3779B97F4A7C15; the low half for even e, the high half for
odd e) are below rint(p * 2**32), and scales what it keeps by 1 / (1 - p).

`own = False`: the operators in elementary torch operations.  `own = True`: gomel_amd's calls.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
GAMMA = 0x9E3779B97F4A7C15
PAGE = 16                       # frames per page of the callers' page tables
MOST = 409600 * 192 * 2         # values of the largest listed cases
FLOOR, TOP = math.log(1e-5), math.log(50.0)


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # an acoustic model that generates one utterance: its next frame goes into the cache and back comes what the cache holds for it
        {"name": "write 1 frame", "op": "write", "n": 1, "bands": 80, "type": "f32", "bits": 8, "group": 0},
        # a batch of 256 utterances generated together, one frame each, in the model's 16-bit type
        {"name": "write 256 frames, 4 bits", "op": "write", "n": 256, "bands": 192, "type": "bf16", "bits": 4, "group": 16},
        # 256 utterances of about 400 frames, written after the spectrograms were made
        {"name": "write 256 utterances", "op": "write", "n": 102400, "bands": 192, "type": "f32", "bits": 8, "group": 0},
        # one rank's share of a corpus, as ToMel's doubles
        {"name": "write a shard, 4 bits", "op": "write", "n": 409600, "bands": 192, "type": "f64", "bits": 4, "group": 32},
        # streaming: 64 utterances get their next frame, the last 16 frames of each are read back for the next piece of audio
        {"name": "write 64, read 64 x 16", "op": "step", "n": 64, "window": 16, "bands": 160, "type": "f16", "bits": 8, "group": 32},
        # one 10 s utterance on its way into FromMel
        {"name": "read 858 frames", "op": "read", "n": 858, "bands": 80, "type": "f32", "bits": 8, "group": 0, "p": 0.0},
        # a training batch of ragged utterances with the input dropout in the same pass
        {"name": "read a batch, dropout", "op": "read", "n": 54912, "bands": 80, "type": "bf16", "bits": 8, "group": 0, "p": 0.1},
        # 256 utterances held in 4 bits, into FromMel's batch
        {"name": "read 256 utterances, 4 bits", "op": "read", "n": 102400, "bands": 192, "type": "f32", "bits": 4, "group": 16, "p": 0.0},
        # one rank's share of a corpus
        {"name": "read a shard", "op": "read", "n": 409600, "bands": 192, "type": "bf16", "bits": 8, "group": 64, "p": 0.0},
        # frames of a small odd-sized step, both directions
        {"name": "dropout 33 x 322, both", "op": "dropout", "n": 33, "bands": 161, "type": "f16", "p": 0.5, "pass": "both"},
        # the training batch's frames, both directions, in the model's type
        {"name": "dropout a batch, both", "op": "dropout", "n": 102400, "bands": 192, "type": "bf16", "p": 0.1, "pass": "both"},
        # the gradient of one rank's share
        {"name": "dropout a shard, backward", "op": "dropout", "n": 409600, "bands": 192, "type": "f32", "p": 0.25, "pass": "backward"},
    ]


def draw(rng):
    op = rng.choice(["write", "write", "read", "read", "step", "dropout", "dropout"])
    bands = rng.choice([80, 160, 192, rng.randint(20, 300), 2 * rng.randint(10, 150) + 1])
    most = 4096 if op == "step" else MOST // (2 * bands)
    c = {"op": op, "n": int(round(math.exp(rng.uniform(0.0, math.log(most))))), "bands": bands, "type": rng.choice(sorted(TYPES))}
    if op == "dropout":
        c["p"], c["pass"] = round(rng.uniform(0.02, 0.6), 3), rng.choice(["forward", "backward", "both"])
        if c["pass"] == "both":
            c["n"] = max(1, c["n"] // 2)
        return c
    c["bits"], c["group"] = rng.choice([8, 4]), rng.choice([0, 8, 16, 32, 64])
    if op == "step":
        c["window"] = rng.choice([1, 4, 16, 32])
    if op == "read":
        c["p"] = rng.choice([0.0, 0.0, round(rng.uniform(0.02, 0.5), 3)])
    return c


def _groups(case):
    return 1 if not case["group"] else -(-case["bands"] // case["group"])


def work(case):
    n, values, size = case["n"], 2 * case["n"] * case["bands"], BYTES[case["type"]]
    if case["op"] == "dropout":
        passes = 2 if case["pass"] == "both" else 1
        return {"bytes": 2 * passes * values * size, "flops": passes * values}
    held = 2 * case["bands"] * case["bits"] / 8 + 8 * _groups(case)     # codes, lo and step of a frame
    if case["op"] == "write":
        return {"bytes": 2 * values * size + n * (held + 8), "flops": 8 * values}
    if case["op"] == "read":
        return {"bytes": values * size + n * (held + 8), "flops": (3 if case["p"] else 2) * values}
    w = case["window"]
    return {"bytes": values * size * (1 + w) + n * (1 + w) * (held + 8), "flops": (8 + 2 * w) * values}


# -------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _frames(case, n, seed, salt=0):
    """Log-mel frames: a spectral slope with resonances and noise per frame, quieter and louder frames, ToMel's floor ln(1e-5) where the
    signal is below it (whole silent frames among them); the second channel is the neighbouring bin's magnitude, close to the first."""
    k, g = case["bands"], _gen(seed, salt)
    band = torch.arange(k, device="cuda", dtype=torch.float32) / k
    level = torch.rand(n, 1, generator=g, device="cuda") * 9.0 - 8.0
    tilt = torch.rand(n, 1, generator=g, device="cuda") * -6.0
    phase = torch.rand(n, 1, generator=g, device="cuda") * 6.28
    x = torch.sin(band * 19.0 + phase).mul_(1.5).add_(band * tilt).add_(level)
    x = x.unsqueeze(2).repeat(1, 1, 2)
    x += torch.randn(x.shape, generator=g, device="cuda").mul_(0.5)
    x.clamp_(FLOOR, TOP)
    if case["type"] == "f64":
        x = x.double()
        x += torch.randn(1, generator=g, device="cuda", dtype=torch.float64) * 1e-3      # values that 32 bits do not hold
        x.clamp_(FLOOR, TOP)
    return x.to(TYPES[case["type"]])


def _slots(count, seed):
    """Where the frames of ragged utterances (about 400 each) stand: pages of 16 frames in any order, the last page of each partly used."""
    rng = np.random.RandomState((seed * 7919 + 17) % (1 << 31))
    lens, left = [], count
    while left > 0:
        lens.append(min(left, int(rng.randint(200, 601))))
        left -= lens[-1]
    pages = [-(-m // PAGE) for m in lens]
    order, at, got = rng.permutation(sum(pages)), 0, []
    for m, p in zip(lens, pages):
        got.append((order[at:at + p, None].astype(np.int64) * PAGE + np.arange(PAGE)).reshape(-1)[:m])
        at += p
    return torch.from_numpy(np.concatenate(got)).cuda(), PAGE * len(order)


def _step_slots(case, seed):
    """Each stream's window of its last frames; the newest one is what the step writes."""
    n, w = case["n"], case["window"]
    per = -(-(w + 7) // PAGE) * PAGE
    rng = np.random.RandomState((seed * 7919 + 29) % (1 << 31))
    table = rng.permutation(n * per // PAGE).reshape(n, -1)
    at = rng.randint(0, per - w + 1, n)[:, None] + np.arange(w)
    read = np.take_along_axis(table, at // PAGE, 1) * PAGE + at % PAGE
    return torch.from_numpy(read.reshape(-1).astype(np.int64)).cuda(), torch.from_numpy(read[:, -1].astype(np.int64).copy()).cuda(), n * per


def _seed64(seed):
    return (seed * 0x2545F4914F6CDD1D + 0x1234567) & (2 ** 64 - 1)


def _inputs(case, seed):
    """What the passes take, whatever computes them."""
    s, n = {"case": dict(case)}, case["n"]
    if case["op"] == "dropout":
        s["x"] = _frames(case, n, seed).reshape(n, -1)
        if case["pass"] != "forward":
            s["dy"] = torch.randn(n, 2 * case["bands"], generator=_gen(seed, 5), device="cuda").to(TYPES[case["type"]])
    elif case["op"] == "write":
        s["x"], (s["slots"], s["held"]) = _frames(case, n, seed), _slots(n, seed)
    elif case["op"] == "read":
        s["slots"], s["held"] = _slots(n, seed)
        s["before"] = _frames(case, n, seed)
    else:
        s["slots"], s["new"], s["held"] = _step_slots(case, seed)
        s["before"], s["x"] = _frames(case, n * case["window"], seed), _frames(case, n, seed, 3)
    s["seed"], s["offset"] = _seed64(seed), (seed % 97) * 2 * case["bands"]
    return s


_handles = {}


def _engine(bands):
    import gomel_amd
    if bands not in _handles:
        m = gomel_amd.NewMel()
        m.NumMels, m.MelFmax, m.Window, m.Resolut, m.Device = bands, 16000, 1280, 4096, 0
        _handles[bands] = m.engine()
    return _handles[bands]


def prepare(case, seed):
    s = _inputs(case, seed)
    n, k = case["n"], case["bands"]
    if case["op"] == "dropout":
        s["p"] = case["p"]
        if own:
            s["engine"] = _engine(k)
            s["y"], s["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        return s
    rows = s["slots"].numel()
    s["out"] = torch.empty(rows, k, 2, dtype=TYPES[case["type"]], device="cuda")
    if own:
        s["cache"] = _engine(k).cache(s["held"], bits=case["bits"], group=case["group"])
        if "before" in s:
            s["cache"].write(s.pop("before"), slots=s["slots"])
    else:
        width = k * 2 if case["bits"] == 8 else k
        s["codes"] = torch.zeros(s["held"], width, dtype=torch.uint8, device="cuda")
        s["lo"] = torch.zeros(s["held"], _groups(case), dtype=torch.float32, device="cuda")
        s["step"] = torch.zeros_like(s["lo"])
        if "before" in s:
            _plain_write(s, s.pop("before"), s["slots"])
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _plain_write(s, x, slots):
    """Quantises x [n][K][2] into the state's codes, lo and step at `slots`; the values that the codes stand for."""
    c, levels = s["case"], 2 ** s["case"]["bits"] - 1
    n, k = x.shape[0], x.shape[1]
    group = c["group"] or k
    count = -(-k // group)
    x = x.double()                                                    # in 64 bits: codes sit next to a border
    room = count * group - k
    low = torch.nn.functional.pad(x, (0, 0, 0, room), value=math.inf) if room else x
    high = torch.nn.functional.pad(x, (0, 0, 0, room), value=-math.inf) if room else x
    lo = low.reshape(n, count, 2 * group).amin(2).float()
    hi = high.reshape(n, count, 2 * group).amax(2).float()
    step = ((hi.double() - lo.double()) / levels).float()
    of = torch.arange(k, device=x.device) // group
    lo_k, step_k = lo[:, of].unsqueeze(2).double(), step[:, of].unsqueeze(2).double()
    q = torch.where(step_k > 0, torch.round((x - lo_k) / step_k), torch.zeros_like(x)).clamp(0, levels)
    codes = q.to(torch.uint8)
    codes = codes.reshape(n, 2 * k) if c["bits"] == 8 else codes[:, :, 0] | (codes[:, :, 1] << 4)
    s["codes"][slots], s["lo"][slots], s["step"][slots] = codes, lo, step
    return (lo_k + q * step_k).to(TYPES[c["type"]])


def _plain_words(seed, offset, count, device):
    """The 32 random bits of the elements offset ... offset + count - 1."""
    def shift(v, b):
        return (v >> b) & ((1 << (64 - b)) - 1)

    def signed(v):
        v &= 2 ** 64 - 1
        return v - 2 ** 64 if v >> 63 else v
    e = torch.arange(offset, offset + count, device=device, dtype=torch.int64)
    z = ((e >> 1) + 1) * signed(GAMMA) + signed(seed)
    z = (z ^ shift(z, 30)) * signed(0xBF58476D1CE4E5B9)
    z = (z ^ shift(z, 27)) * signed(0x94D049BB133111EB)
    z = z ^ shift(z, 31)
    return torch.where((e & 1).bool(), shift(z, 32), z & 0xFFFFFFFF)


def _plain_dropout(x, p, seed, offset):
    kept = _plain_words(seed, offset, x.numel(), x.device).reshape(x.shape) >= int(round(p * 2 ** 32))
    wide = x if x.dtype == torch.float64 else x.float()
    return torch.where(kept, wide * (1.0 / (1.0 - p)), torch.zeros_like(wide)).to(x.dtype)


def _plain_read(s, slots, p):
    c = s["case"]
    k, wide = c["bands"], torch.float64 if c["type"] == "f64" else torch.float32
    codes = s["codes"][slots]
    q = codes.reshape(-1, k, 2) if c["bits"] == 8 else torch.stack((codes & 15, codes >> 4), 2)
    of = torch.arange(k, device=codes.device) // (c["group"] or k)
    v = s["lo"][slots][:, of].unsqueeze(2).to(wide) + q.to(wide) * s["step"][slots][:, of].unsqueeze(2).to(wide)
    if p:
        kept = _plain_words(s["seed"], s["offset"], v.numel(), v.device).reshape(v.shape) >= int(round(p * 2 ** 32))
        v = torch.where(kept, v * (1.0 / (1.0 - p)), torch.zeros_like(v))
    return v.to(TYPES[c["type"]])


def run(state):
    s, c = state, state["case"]
    if c["op"] == "dropout":
        got = {}
        if own:
            if c["pass"] != "backward":
                got["y"] = s["engine"].dropout(s["x"], s["p"], s["seed"], s["offset"], out=s["y"])
            if c["pass"] != "forward":
                got["dx"] = s["engine"].dropout_backward(s["dy"], s["p"], s["seed"], s["offset"], out=s["dx"])
            return got
        if c["pass"] != "backward":
            got["y"] = _plain_dropout(s["x"], s["p"], s["seed"], s["offset"])
        if c["pass"] != "forward":
            got["dx"] = _plain_dropout(s["dy"], s["p"], s["seed"], s["offset"])
        return got
    if c["op"] == "write":
        return s["cache"].write(s["x"], slots=s["slots"], values=s["out"]) if own else _plain_write(s, s["x"], s["slots"])
    if c["op"] == "read":
        return s["cache"].read(s["out"], slots=s["slots"], p=c["p"], seed=s["seed"], offset=s["offset"]) if own else _plain_read(s, s["slots"], c["p"])
    if own:
        s["cache"].write(s["x"], slots=s["new"])
        return s["cache"].read(s["out"], slots=s["slots"])
    _plain_write(s, s["x"], s["new"])
    return _plain_read(s, s["slots"], 0.0)


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def _stands_for(x, bits, group):
    """What frames x [n][K][2] (float64) read as, frame by frame and group by group of the definition."""
    out, top = torch.empty_like(x), float(2 ** bits - 1)
    k = x.shape[1]
    for b in range(0, k, group or k):
        v = x[:, b:b + (group or k)]
        a = v.amin((1, 2), keepdim=True).float().double()
        d = ((v.amax((1, 2), keepdim=True).float().double() - a) / top).float().double()
        q = ((v - a) / torch.where(d == 0, torch.ones_like(d), d)).round().clamp_(0.0, top)
        out[:, b:b + (group or k)] = torch.addcmul(a.expand_as(v), q, d.expand_as(v))
    return out


def _kept(p, seed, offset, count):
    """Which of `count` elements dropout keeps (numpy, unsigned 64-bit arithmetic, one word for two elements)."""
    first = offset // 2
    z = np.arange(first + 1, (offset + count + 1) // 2 + 1, dtype=np.uint64)
    z *= np.uint64(GAMMA)
    z += np.uint64(seed)
    for by, m in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
        z ^= z >> np.uint64(by)
        z *= np.uint64(m)
    z ^= z >> np.uint64(31)
    halves = z.view(np.uint32)                                        # little endian: the low half first
    at = offset - 2 * first
    return halves[at:at + count] >= np.uint64(int(round(p * 2 ** 32)))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "dropout":
        keep = torch.from_numpy(_kept(case["p"], s["seed"], s["offset"], s["x"].numel())).cuda().reshape(s["x"].shape)
        names = {"forward": (("y", "x"),), "backward": (("dx", "dy"),), "both": (("y", "x"), ("dx", "dy"))}[case["pass"]]
        return {to: (s[of].double() / (1.0 - case["p"])).masked_fill_(~keep, 0.0) for to, of in names}
    if case["op"] == "write":
        return _stands_for(s["x"].double(), case["bits"], case["group"])
    v = _stands_for(s["before"].double(), case["bits"], case["group"])
    if case["op"] == "step":
        n = case["n"]
        v.reshape(n, case["window"], case["bands"], 2)[:, -1] = _stands_for(s["x"].double(), case["bits"], case["group"])
    elif case["p"]:
        keep = torch.from_numpy(_kept(case["p"], s["seed"], s["offset"], v.numel())).cuda().reshape(v.shape)
        v = (v / (1.0 - case["p"])).masked_fill_(~keep, 0.0)
    return v
