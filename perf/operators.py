"""Cases of the block-scaled 4-bit operators: quantisation, its inverse, and the product of two such matrices.

A matrix of rows x cols is held as 4-bit floats (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a
byte, low nibble first, every row padded with zero codes to a whole number of 32, and one scale for each block of
neighbours in a row:

  mxfp4   blocks of 32, scale = 2^(floor(log2(max|v|)) - 2) held as an exponent byte (e8m0)
  nvfp4   blocks of 16, scale = max|v| / (6 t) rounded to e4m3, and one 32-bit scale t for the whole matrix, which is
          the smallest power of two that keeps every block's scale within e4m3 (or given by the caller)

and code = v / (scale t) rounded to e2m1, ties to even, at most 6.  The scales lie in rows ("rows") or in the tiles of
128 rows x 4 blocks that the product reads ("tiled").  The product is A B^T of two such matrices.

`own` false computes all of this with elementary torch operations; `own` true makes the library's calls.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a token's activations on their way into a 4-bit layer, the calibrated scale given: latency counts
        dict(name="quantize_token", op="quantize", format="nvfp4", layout="tiled", dtype="f16", rows=1, cols=4096, pad=0, given=True),
        # one feed-forward weight of the 7B-shaped model, scales in rows as a blob stores them
        dict(name="quantize_weights", op="quantize", format="mxfp4", layout="rows", dtype="f16", rows=11008, cols=4096, pad=0, given=False),
        # the output head of that model from 32-bit masters; the matrix's own scale is found first
        dict(name="quantize_head", op="quantize", format="nvfp4", layout="tiled", dtype="f32", rows=32000, cols=4096, pad=0, given=False),
        # rows that end inside a block, cut out of a wider buffer whose rows no vector load can rely on
        dict(name="quantize_ragged", op="quantize", format="mxfp4", layout="tiled", dtype="bf16", rows=1777, cols=1003, pad=7, given=False),
        # a stored weight read back for a layer that runs in 16 bits
        dict(name="dequantize_weights", op="dequantize", format="mxfp4", layout="rows", dtype="f16", rows=11008, cols=4096),
        # a small odd matrix in the product's layout, read back to 32 bits
        dict(name="dequantize_ragged", op="dequantize", format="nvfp4", layout="tiled", dtype="f32", rows=333, cols=2005),
        # one token through a feed-forward weight: activations quantised, then the product
        dict(name="linear_token", op="linear", format="nvfp4", dtype="f16", m=1, n=11008, k=4096),
        # a decode batch through the weight that leads back
        dict(name="linear_tokens", op="linear", format="mxfp4", dtype="bf16", m=16, n=4096, k=11008),
        # a short prompt through an attention projection, one row more than a round number
        dict(name="linear_prompt", op="linear", format="mxfp4", dtype="f16", m=257, n=4096, k=4096),
        # a prefill chunk with its activations already in 4 bits
        dict(name="matmul_prefill", op="matmul", format="mxfp4", dtype="f16", m=2048, n=11008, k=4096),
        # a whole calibration batch: bound by the tensor cores
        dict(name="matmul_batch", op="matmul", format="nvfp4", dtype="bf16", m=8192, n=4096, k=11008),
        # nothing is a round number, and the sums are wanted in 32 bits
        dict(name="matmul_ragged", op="matmul", format="nvfp4", dtype="f32", m=77, n=515, k=1003),
    ]


def _size(rng, top):
    return min(top, max(1, round(math.exp(rng.uniform(0.0, math.log(top))))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "linear", "matmul"])
    case = dict(op=op, format=rng.choice(["mxfp4", "nvfp4"]), dtype=rng.choice(["f16", "bf16", "f32"]))
    if op in ("quantize", "dequantize"):
        case.update(layout=rng.choice(["rows", "tiled"]), rows=_size(rng, 32000), cols=_size(rng, 4096))
        if op == "quantize":
            case.update(pad=rng.choice([0, 0, 8, rng.randrange(1, 32)]), given=rng.random() < 0.5)
        return case
    if op == "linear":
        case["dtype"] = rng.choice(["f16", "bf16"])
    while True:
        m, n, k = _size(rng, 8192), _size(rng, 11008), _size(rng, 11008)
        if m * n * k <= 8192 * 4096 * 11008:
            return dict(case, m=m, n=n, k=k)


def _held(rows, cols, fmt):
    """Bytes of a matrix's codes and scales, without padding."""
    return rows * ((cols + 1) // 2) + rows * -(-cols // BLOCK[fmt])


def work(case):
    f = case["format"]
    if case["op"] in ("quantize", "dequantize"):
        n, es = case["rows"] * case["cols"], BYTES[case["dtype"]]
        held = _held(case["rows"], case["cols"], f)
        # quantize: the input, the codes and scales, and the values that they stand for; dequantize: codes, scales, values
        return {"bytes": held + n * es * (2 if case["op"] == "quantize" else 1), "flops": 2 * n}
    m, n, k, es = case["m"], case["n"], case["k"], BYTES[case["dtype"]]
    a = m * k * es if case["op"] == "linear" else _held(m, k, f)
    return {"bytes": a + _held(n, k, f) + m * n * es, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------- layouts
def _pitch(cols):
    return -(-cols // 32) * 16  # bytes of a row of codes


def _nblk(cols, fmt):
    return -(-cols // BLOCK[fmt])


def _lay(scales, layout):
    """Scales [rows, blocks] -> the bytes as they are stored; what pads a tile is 0."""
    if layout == "rows":
        return scales.contiguous()
    r, b = scales.shape
    R, B = -(-r // 128), -(-b // 4)
    full = torch.zeros(R * 128, B * 4, dtype=scales.dtype, device=scales.device)
    full[:r, :b] = scales
    # row = tile * 128 + quarter * 32 + line, block = chunk * 4 + k; a tile's chunk is 512 bytes: [line][quarter][k]
    return full.view(R, 4, 32, B, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _unlay(stored, rows, blocks, layout):
    if layout == "rows":
        return stored.view(rows, blocks)
    R, B = -(-rows // 128), -(-blocks // 4)
    return stored.view(R, B, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(R * 128, B * 4)[:rows, :blocks]


# --------------------------------------------------------------------------- plain form, 32 bits
def _blocks(x, fmt):
    """x [rows, cols] -> 32-bit [rows, blocks, block], zeros behind the last column."""
    r, c = x.shape
    b = BLOCK[fmt]
    x = x.float()
    if c % b:
        x = torch.cat([x, x.new_zeros(r, b - c % b)], 1)
    return x.view(r, -1, b)


def _two_to(e):
    """2^e in 32 bits from its exponent field, e in -126 .. 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _power_above(a):
    """The smallest power of two t with a <= 2688 t: 2688 = 6 * 448 = 0.65625 * 2^12."""
    m, e = torch.frexp(a)
    e = torch.where(m <= 0.65625, e - 12, e - 11).clamp(-126, 127)
    return torch.where(a > 0, _two_to(e), torch.ones_like(a))


def _codes(q):
    """|q| -> index into 0, 0.5, 1, 1.5, 2, 3, 4, 6: nearest, ties to the even index."""
    q = q.abs()
    return ((q > 0.25).to(torch.uint8) + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5) + (q > 5.0))


def _quantized(x, fmt, t):
    """codes [rows, blocks, block] (sign in bit 3), stored scales [rows, blocks] (uint8), factor of every block."""
    v = _blocks(x, fmt)
    top = v.abs().amax(2)
    if fmt == "mxfp4":
        e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp(-127, 127)
        held = (e + 127).to(torch.uint8)
        q = v * _two_to(-e).unsqueeze(2)
        factor = _two_to(e + 1) * 0.5
    else:
        s = (top / (6.0 * t)).clamp(max=448.0).to(torch.float8_e4m3fn)
        held = s.view(torch.uint8)
        factor = s.float() * t
        q = torch.where(factor.unsqueeze(2) > 0, v / factor.unsqueeze(2), torch.zeros_like(v))
    return _codes(q) | ((v < 0).to(torch.uint8) << 3), held, factor


_MAGNITUDE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _table(device, dtype=torch.float32):
    return torch.tensor(_MAGNITUDE + tuple(-m for m in _MAGNITUDE), dtype=dtype, device=device)


def _pack(codes, cols):
    """codes [rows, blocks, block] -> bytes [rows, pitch]."""
    r = codes.shape[0]
    flat = torch.zeros(r, 2 * _pitch(cols), dtype=torch.uint8, device=codes.device)
    flat[:, :cols] = codes.view(r, -1)[:, :cols]
    return flat[:, 0::2] | (flat[:, 1::2] << 4)


def _scales_of(held, fmt):
    return held.view(torch.float8_e8m0fnu if fmt == "mxfp4" else torch.float8_e4m3fn)


def _values(m, dtype=torch.float32):
    """The values that a held matrix stands for."""
    fmt, rows, cols = m["format"], m["rows"], m["cols"]
    both = torch.stack([m["codes"] & 15, m["codes"] >> 4], 2).view(rows, -1)
    scale = _scales_of(_unlay(m["scales"], rows, _nblk(cols, fmt), m["layout"]).contiguous(), fmt).to(dtype)
    if fmt == "nvfp4":
        scale = scale * m["tensor_scale"][0].to(dtype)
    v = _table(both.device, dtype)[both[:, :_nblk(cols, fmt) * BLOCK[fmt]].int()]
    return (v.view(rows, -1, BLOCK[fmt]) * scale.unsqueeze(2)).view(rows, -1)[:, :cols]


def _hold(x, fmt, layout, t=None):
    """A held matrix made from x: what a program has of its weights."""
    t = (_power_above(x.abs().amax().float()) if t is None else t) if fmt == "nvfp4" else None
    codes, held, _ = _quantized(x, fmt, t)
    m = dict(format=fmt, layout=layout, rows=x.shape[0], cols=x.shape[1], codes=_pack(codes, x.shape[1]), scales=_lay(held, layout))
    if fmt == "nvfp4":
        m["tensor_scale"] = torch.stack([t, x.abs().amax().float()])
    return m


# --------------------------------------------------------------------------- inputs
def _activations(rows, cols, dtype, g):
    """Normal values whose columns differ in size, a few of them far larger, as activations are."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))
    x[:, torch.rand(cols, device="cuda", generator=g) < 0.005] *= 8.0
    return x.to(dtype)


def _weights(rows, cols, dtype, g):
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= 0.02 * torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))
    return x.to(dtype)


_library = None


def _lib():
    """The library's handle, on torch's stream: made once, as a program does."""
    global _library
    if _library is None:
        from npu_plugin_b200 import _cabi, const, mx
        backend = const.CudaBackend(torch.cuda.current_device())
        backend.set_stream(torch.cuda.current_stream().cuda_stream)
        codes = {"f16": _cabi.F16, "bf16": _cabi.BF16, "f32": _cabi.F32}
        formats = {"mxfp4": _cabi.MXFP4, "nvfp4": _cabi.NVFP4}
        layouts = {"rows": _cabi.MX_SCALES_ROWS, "tiled": _cabi.MX_SCALES_TILED}
        _library = (backend, mx, codes, formats, layouts)
    return _library


def _matrix(m):
    """The library's descriptor of a held matrix."""
    _, mx, _, formats, layouts = _lib()
    t = m.get("tensor_scale")
    return mx.MxMatrix(formats[m["format"]], m["rows"], m["cols"], m["codes"].data_ptr(), m["scales"].data_ptr(),
                       tensor_scale=None if t is None else t.data_ptr(), layout=layouts[m["layout"]])


def _empty(fmt, layout, rows, cols, t):
    """Buffers for a matrix to be quantised into."""
    blocks = _nblk(cols, fmt)
    n = (rows, blocks) if layout == "rows" else (-(-rows // 128) * -(-blocks // 4) * 512,)
    m = dict(format=fmt, layout=layout, rows=rows, cols=cols,
             codes=torch.zeros(rows, _pitch(cols), dtype=torch.uint8, device="cuda"),
             scales=torch.zeros(n, dtype=torch.uint8, device="cuda"))
    if fmt == "nvfp4":
        m["tensor_scale"] = torch.zeros(2, device="cuda") if t is None else torch.stack([t, t])
    return m


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    fmt, dtype = case["format"], DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        make = _activations if case["given"] else _weights
        s["x"] = make(rows, cols + case["pad"], dtype, g)[:, :cols]
        s["t"] = _power_above(s["x"].abs().amax().float()) if fmt == "nvfp4" and case["given"] else None
        if own:
            s["q"] = _empty(fmt, case["layout"], rows, cols, s["t"])
            s["matrix"] = _matrix(s["q"])
            s["values"] = torch.empty(rows, cols, dtype=dtype, device="cuda")
    elif case["op"] == "dequantize":
        s["q"] = _hold(_weights(case["rows"], case["cols"], torch.float32, g), fmt, case["layout"])
        if fmt == "nvfp4":
            s["q"]["tensor_scale"] = s["q"]["tensor_scale"] * 0.7  # a stored scale need not be a power of two
        if own:
            s["matrix"] = _matrix(s["q"])
            s["values"] = torch.empty(case["rows"], case["cols"], dtype=dtype, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = _activations(m, k, dtype if case["op"] == "linear" else torch.float32, g)
        t = _power_above(x.abs().amax().float()) if fmt == "nvfp4" else None
        s["b"] = _hold(_weights(n, k, torch.float32, g), fmt, "tiled")
        if case["op"] == "linear":
            s["x"], s["t"] = x, t
            if own:
                s["a"] = _empty(fmt, "tiled", m, k, t)
        else:
            s["a"] = _hold(x, fmt, "tiled", t)
        if own:
            s["ma"], s["mb"] = _matrix(s["a"]), _matrix(s["b"])
            s["out"] = torch.empty(m, n, dtype=dtype, device="cuda")
    return s


# --------------------------------------------------------------------------- one pass
def _answer(s, held, values, t):
    out = {"scales": _scales_of(held, s["format"]), "values": values}
    if s["format"] == "nvfp4" and not s["given"]:
        out["tensor_scale"] = t
    return out


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    backend, _, codes, _, _ = _lib()
    dt = codes[s["dtype"]]
    if s["op"] == "quantize":
        backend.mx_quantize(s["x"].data_ptr(), dt, s["x"].stride(0), s["matrix"], tensor_scale_given=s["given"],
                            values=s["values"].data_ptr(), values_ld=s["cols"])
        return _answer(s, s["q"]["scales"], s["values"], s["q"].get("tensor_scale"))
    if s["op"] == "dequantize":
        backend.mx_dequantize(s["matrix"], s["values"].data_ptr(), dt, s["cols"])
        return {"values": s["values"]}
    if s["op"] == "linear":
        backend.mx_quantize(s["x"].data_ptr(), dt, s["x"].stride(0), s["ma"], tensor_scale_given=True)
    backend.mx_matmul(s["ma"], s["mb"], s["out"].data_ptr(), dt, s["n"])
    return {"out": s["out"]}


def _run_plain(s):
    fmt, dtype = s["format"], DTYPES[s["dtype"]]
    if s["op"] == "quantize":
        x, t, top = s["x"], s["t"], None
        if fmt == "nvfp4" and t is None:
            top = x.abs().amax().float()
            t = _power_above(top)
        codes, held, factor = _quantized(x, fmt, t)
        values = (_table(x.device)[codes.int()] * factor.unsqueeze(2)).view(x.shape[0], -1)[:, :x.shape[1]].to(dtype)
        return _answer(s, _lay(held, s["layout"]), values, None if top is None else torch.stack([t, top]))
    if s["op"] == "dequantize":
        return {"values": _values(s["q"]).to(dtype)}
    if s["op"] == "linear":
        codes, _, factor = _quantized(s["x"], fmt, s["t"])
        a = (_table(codes.device)[codes.int()] * factor.unsqueeze(2)).view(s["m"], -1)[:, :s["k"]]
    else:
        a = _values(s["a"])
    return {"out": torch.matmul(a, _values(s["b"]).t()).to(dtype)}


# --------------------------------------------------------------------------- the definition in 64 bits
def _nearest(q):
    """|q| to the nearest e2m1 magnitude, ties to the even one: borders at the middles, those whose upper neighbour is
    even taken one step lower so that the tie falls up."""
    down = lambda b: math.nextafter(b, 0.0)
    borders = torch.tensor([0.25, down(0.75), 1.25, down(1.75), 2.5, down(3.5), 5.0], dtype=torch.float64, device=q.device)
    return torch.tensor(_MAGNITUDE, dtype=torch.float64, device=q.device)[torch.bucketize(q.abs(), borders)]


def _floor_power(a):
    """2^floor(log2 a) of positive 64-bit values: the number with its fraction bits cleared, so that no tie is lost to a logarithm's last bit."""
    return (a.view(torch.int64) & (2047 << 52)).view(torch.float64)


def _exact_quantized(x, fmt, t):
    """(values, scales) of x in 64 bits: the scale of every block, then the nearest code times it."""
    r, c = x.shape
    b = BLOCK[fmt]
    v = torch.nn.functional.pad(x.double(), (0, -c % b)).unflatten(1, (-1, b))
    top = v.abs().amax(2)
    if fmt == "mxfp4":
        s = _floor_power(top.clamp(min=2.0 ** -125)) / 4.0
        s = torch.where(top >= 2.0 ** -125, s, torch.full_like(s, 2.0 ** -127))
        f = s
    else:
        w = (top / (6.0 * t)).clamp(max=448.0)
        step = _floor_power(w.clamp(min=2.0 ** -6)) / 8.0
        s = torch.round(w / step) * step
        f = s * t
    q = torch.where(f.unsqueeze(2) > 0, v / f.unsqueeze(2), 0.0)
    return (torch.sign(v) * _nearest(q) * f.unsqueeze(2)).flatten(1)[:, :c], s


def _exact_scale(top):
    """The smallest power of two t with top <= 2688 t."""
    return 2.0 ** max(-126, math.ceil(math.log2(top / 2688.0))) if top > 0 else 1.0


def _place(r, b, blocks):
    """Where the tiled layout keeps the scale of row r, block b."""
    return ((r // 128) * -(-blocks // 4) + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def _exact_held(m):
    """The values of a held matrix, byte by byte, in 64 bits."""
    rows, cols, fmt = m["rows"], m["cols"], m["format"]
    r = torch.arange(rows, device="cuda").unsqueeze(1)
    b = torch.arange(_nblk(cols, fmt), device="cuda").unsqueeze(0)
    if m["layout"] == "rows":
        at = r * _nblk(cols, fmt) + b
    else:
        at = _place(r, b, _nblk(cols, fmt))
    byte = m["scales"].view(-1)[at].long()
    if fmt == "mxfp4":
        scale = ((byte - 127 + 1023) << 52).view(torch.float64)
    else:
        e, f = byte >> 3 & 15, (byte & 7).double()
        scale = torch.where(e > 0, ((e - 7 + 1023) << 52).view(torch.float64) * (1.0 + f / 8.0), f * 2.0 ** -9) * m["tensor_scale"][0].double()
    c = torch.arange(cols, device="cuda")
    code = m["codes"][:, c // 2].int() >> (4 * (c % 2)).int() & 15
    mag = torch.tensor(_MAGNITUDE, dtype=torch.float64, device="cuda")[code & 7]
    return torch.where(code > 7, -mag, mag) * scale[:, c // BLOCK[fmt]]


def exact(case, seed):
    s = prepare(case, seed)
    fmt = s["format"]
    if s["op"] == "quantize":
        top = float(s["x"].abs().max())
        t = 1.0 if fmt == "mxfp4" else float(s["t"]) if s["given"] else _exact_scale(top)
        parts = [_exact_quantized(p, fmt, t) for p in s["x"].split(4096)]  # a few rows at a time: 64 bits are wide
        values, scales = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        if s["layout"] == "tiled":
            r, b = (torch.arange(n, device="cuda") for n in scales.shape)
            stored = torch.full((-(-len(r) // 128) * -(-len(b) // 4) * 512,), 2.0 ** -127 if fmt == "mxfp4" else 0.0,
                                dtype=torch.float64, device="cuda")
            stored[_place(r.unsqueeze(1), b.unsqueeze(0), len(b))] = scales
            scales = stored
        out = {"scales": scales, "values": values}
        if fmt == "nvfp4" and not s["given"]:
            out["tensor_scale"] = torch.tensor([t, top], dtype=torch.float64, device="cuda")
        return out
    if s["op"] == "dequantize":
        return {"values": _exact_held(s["q"])}
    if s["op"] == "linear":
        a, _ = _exact_quantized(s["x"], fmt, 1.0 if fmt == "mxfp4" else float(s["t"]))
    else:
        a = _exact_held(s["a"])
    return {"out": a @ _exact_held(s["b"]).t()}
