"""Block-scaled 4-bit matrices: quantisation and its inverse against a 64-bit oracle, byte for byte, and the refusals
of their entry points.  The refusals run without a device: every argument is checked before the context is."""
import ctypes as C

import numpy as np
import pytest

import mx_oracle as O
from npu_plugin_b200 import _cabi as A
from npu_plugin_b200 import mx

torch = pytest.importorskip("torch")

FORMATS = [A.MXFP4, A.NVFP4]
LAYOUTS = [A.MX_SCALES_ROWS, A.MX_SCALES_TILED]
TYPES = {A.F16: torch.float16, A.BF16: torch.bfloat16, A.F32: torch.float32}
CANARY = 0xA5


# --------------------------------------------------------------------------- host side
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(0, 0), (1, 1), (1, 32), (127, 33), (128, 64), (129, 4096), (5, 1003)])
def test_sizes(fmt, rows, cols):
    blocks = -(-cols // O.BLOCK[fmt])
    assert mx.sizes(fmt, rows, cols, A.MX_SCALES_ROWS) == (-(-cols // 32) * 16, rows * -(-cols // 32) * 16, rows * blocks)
    tiles = -(-rows // 128) * -(-blocks // 4)
    assert mx.sizes(fmt, rows, cols) == (-(-cols // 32) * 16, rows * -(-cols // 32) * 16, tiles * 512)


def matrix(**kw):
    a = dict(fmt=A.NVFP4, rows=64, cols=64, codes=0x10000, scales=0x20000, tensor_scale=0x30000)
    a.update(kw)
    return mx.MxMatrix(**a)


def refused(call, *args):
    lib = A.load()
    assert getattr(lib, call)(None, *args) == A.ERR_INVALID
    return lib.b200c_last_error().decode()


QUANTIZE = dict(src=0x100000, dtype=A.F16, ld=64, values=None, values_ld=0, flags=0)


@pytest.mark.parametrize("change,said", [
    (dict(), "null context"),
    (dict(dtype=A.F64), "element type"), (dict(dtype=A.SI8), "element type"),
    (dict(ld=63), "fewer elements"), (dict(src=None), "source: null"), (dict(src=0x100001), "not aligned"),
    (dict(values=0x200000, values_ld=63), "values: fewer"), (dict(values=0x200001, values_ld=64), "values: not aligned"),
    (dict(values=0x100000, values_ld=64), "overlaps source"), (dict(values=0x10000, values_ld=64), "overlaps codes"),
    (dict(src=0x10040), "codes overlaps source"), (dict(src=0x20000), "scales overlaps source"),
    (dict(flags=2), "unknown flags"), (dict(ld=1 << 60), "too large"),
    (dict(m=dict(fmt=3)), "format"), (dict(m=dict(layout=2)), "layout"), (dict(m=dict(rows=-1)), "negative"),
    (dict(m=dict(cols=1 << 31)), "too large"), (dict(m=dict(ld=16)), "multiple of 16"), (dict(m=dict(ld=40)), "multiple of 16"),
    (dict(m=dict(codes=None)), "null pointer"), (dict(m=dict(scales=None)), "null pointer"),
    (dict(m=dict(codes=0x10008)), "codes have to be 16-byte"), (dict(m=dict(scales=0x20004)), "tiled scales"),
    (dict(m=dict(tensor_scale=None)), "needs a tensor scale"), (dict(m=dict(tensor_scale=0x30002)), "tensor scale is not"),
    (dict(m=dict(scales=0x10400)), "codes overlaps scales"), (dict(m=dict(tensor_scale=0x10000)), "overlaps tensor scale"),
    (dict(m=dict(fmt=A.MXFP4), flags=A.MX_SCALE_GIVEN), "no tensor scale"),
])
def test_quantize_refusals(change, said):
    a = dict(QUANTIZE, **{k: v for k, v in change.items() if k != "m"})
    kw = change.get("m", {})
    kw.setdefault("ld", 32)
    m = matrix(**kw)
    assert said in refused("b200c_mx_quantize", a["src"], a["dtype"], a["ld"], C.byref(m.c), a["values"], a["values_ld"], a["flags"])


@pytest.mark.parametrize("change,said", [
    (dict(), "null context"), (dict(dtype=A.UI8), "element type"), (dict(ld=60), "fewer elements"), (dict(out=None), "output: null"),
    (dict(out=0x10040), "overlaps codes"), (dict(out=0x30000), "overlaps tensor scale"),
    (dict(m=dict(fmt=0)), "format"), (dict(m=dict(ld=0)), "multiple of 16"), (dict(m=dict(tensor_scale=None)), "needs a tensor scale"),
])
def test_dequantize_refusals(change, said):
    a = dict(out=0x100000, dtype=A.F16, ld=64)
    a.update({k: v for k, v in change.items() if k != "m"})
    kw = change.get("m", {})
    kw.setdefault("ld", 32)
    m = matrix(**kw)
    assert said in refused("b200c_mx_dequantize", C.byref(m.c), a["out"], a["dtype"], a["ld"])


def test_null_descriptors_are_refused():
    assert "null descriptor" in refused("b200c_mx_quantize", 0x1000, A.F16, 8, None, None, 0, 0)
    assert "null descriptor" in refused("b200c_mx_dequantize", None, 0x1000, A.F16, 8)


def test_oracle_rounds_to_the_nearest_code():
    assert O.e2m1(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 100.0, -0.3, -0.0])).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 9, 8]
    assert O.e4m3(np.array([0.0, 448.0, 1.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])).tolist() == [0, 126, 56, 0, 2, 88, 90]


# --------------------------------------------------------------------------- device side
class Held:
    """Buffers of a matrix on the device, each with canary bytes behind it."""

    def __init__(self, fmt, rows, cols, layout, extra_ld=0, t=None):
        self.fmt, self.rows, self.cols, self.layout = fmt, rows, cols, layout
        pitch, _, nscale = mx.sizes(fmt, rows, cols, layout)
        self.pitch, self.ld, self.nscale = pitch, pitch + extra_ld, nscale
        self.codes = torch.full((rows * self.ld + 64,), CANARY, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((nscale + 64,), CANARY, dtype=torch.uint8, device="cuda")
        self.tensor = torch.tensor([t if t is not None else -1.0, -1.0], device="cuda") if fmt == A.NVFP4 else None
        self.m = mx.MxMatrix(fmt, rows, cols, self.codes.data_ptr(), self.scales.data_ptr(),
                             None if self.tensor is None else self.tensor.data_ptr(), ld=self.ld, layout=layout)

    def load(self, q, extra_noise=False):
        """The oracle's codes and scales."""
        self.codes[:self.rows * self.ld].view(self.rows, self.ld)[:, :self.pitch] = torch.from_numpy(O.pack(q["codes"])).cuda()
        self.scales[:self.nscale] = torch.from_numpy(O.lay(q["scales"], self.layout)).cuda()
        if self.tensor is not None:
            self.tensor[0] = float(q["t"])
        return self

    def check(self, q):
        """Every byte as the oracle has it, and nothing written that is not the matrix's."""
        codes = self.codes.cpu().numpy()
        body = codes[:self.rows * self.ld].reshape(self.rows, self.ld) if self.rows else codes[:0].reshape(0, max(self.ld, 1))
        np.testing.assert_array_equal(body[:, :self.pitch], O.pack(q["codes"]))
        assert (body[:, self.pitch:] == CANARY).all() and (codes[self.rows * self.ld:] == CANARY).all()
        scales = self.scales.cpu().numpy()
        np.testing.assert_array_equal(scales[:self.nscale], O.lay(q["scales"], self.layout))
        assert (scales[self.nscale:] == CANARY).all()


@pytest.fixture
def dev(gpu):
    """The backend on torch's current stream, so that tests order their work as torch does."""
    gpu.set_stream(torch.cuda.current_stream().cuda_stream)
    yield gpu
    torch.cuda.synchronize()
    gpu.set_stream(None)


def awkward(rows, cols, dtype, seed, special=True):
    """Values over many magnitudes with ties, zeros of both signs, whole zero blocks, and (special) NaN, infinities,
    the type's largest and smallest values."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 6, (rows, 1))
    ties = rng.integers(-24, 25, (rows, cols)) / 4.0
    x = np.where(rng.random((rows, cols)) < 0.3, ties, x)
    x[rng.random((rows, cols)) < 0.05] = -0.0
    if cols > 40:
        x[rows // 2, 7:40] = 0.0
    t = torch.from_numpy(x).to(TYPES[dtype])
    if special and rows > 2 and cols > 70:
        info = torch.finfo(TYPES[dtype])
        t[0, 3], t[1, 40], t[1, 70], t[2, 64] = float("nan"), float("inf"), -float("inf"), info.tiny
        t[-1, :32] = info.smallest_normal / 4  # subnormal numbers only
    return t


def put(t, pad):
    """On the device inside a wider buffer whose other columns are NaN; offset by `pad` elements from its start."""
    rows, cols = t.shape
    wide = torch.full((rows, cols + 2 * pad), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, pad:pad + cols] = t.cuda()
    return wide[:, pad:pad + cols]


SHAPES = [(1, 1), (1, 16), (1, 31), (3, 33), (5, 100), (129, 96), (130, 515), (2, 4100), (1, 11008), (700, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize(dev, fmt, dtype, rows, cols):
    x = awkward(rows, cols, dtype, rows * 7 + cols)
    q = O.quantize(x.double().numpy(), fmt)
    for layout, pad, extra in ((A.MX_SCALES_ROWS, 0, 0), (A.MX_SCALES_TILED, 8, 16), (A.MX_SCALES_TILED, 3, 48)):
        src = put(x, pad)
        h = Held(fmt, rows, cols, layout, extra)
        values = torch.full((rows, cols + pad), 7.0, dtype=x.dtype, device="cuda")
        dev.mx_quantize(src.data_ptr(), dtype, src.stride(0), h.m, values=values.data_ptr(), values_ld=values.stride(0))
        h.check(q)
        # code * d has at most 24 + 2 bits: 32-bit rounding, then the type's
        want = torch.from_numpy(q["values"].astype(np.float32)).to(x.dtype)
        assert torch.equal(values[:, :cols].cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
        assert (values[:, cols:] == 7.0).all()
        if fmt == A.NVFP4:
            assert h.tensor.tolist() == [float(q["t"]), float(q["top"])]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dtype,rows,cols", [(A.NVFP4, A.BF16, 1300, 4099), (A.MXFP4, A.F32, 1300, 4096), (A.NVFP4, A.F16, 1300, 4128),
                                                 (A.MXFP4, A.F16, 1300, 3999), (A.NVFP4, A.F32, 20000, 250), (A.NVFP4, A.BF16, 40000, 130),
                                                 (A.MXFP4, A.BF16, 9001, 600)])
def test_large_matrices(dev, fmt, dtype, rows, cols):
    """Enough rows for the kernels' form with several pieces of a row per thread, aligned and not, and back."""
    x = awkward(rows, cols, dtype, cols)
    q = O.quantize(x.double().numpy(), fmt)
    want = torch.from_numpy(q["values"].astype(np.float32)).to(x.dtype).nan_to_num(nan=12345.0)
    for pad in (0, 5):
        src = put(x, pad)
        h = Held(fmt, rows, cols, A.MX_SCALES_TILED)
        values = torch.full((rows, cols + pad), 7.0, dtype=x.dtype, device="cuda")
        dev.mx_quantize(src.data_ptr(), dtype, src.stride(0), h.m, values=values.data_ptr(), values_ld=values.stride(0))
        h.check(q)
        assert torch.equal(values[:, :cols].cpu().nan_to_num(nan=12345.0), want) and (values[:, cols:] == 7.0).all()
        back = torch.full((rows, cols + pad), 7.0, dtype=x.dtype, device="cuda")
        dev.mx_dequantize(h.m, back.data_ptr(), dtype, back.stride(0))
        assert torch.equal(back[:, :cols].cpu().nan_to_num(nan=12345.0), want) and (back[:, cols:] == 7.0).all()


def read_once_input(kind, dtype, rows, cols):
    """More than 128 MB, of which a part may say little about the rest."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    if kind == "outlier":
        x[1, cols // 2] = 3000.0
    elif kind == "few rows":
        keep = x[[1, 778, rows - 1]] * 2.0 ** -5
        x.zero_()
        x[[1, 778, rows - 1]] = keep
    elif kind == "steep":
        x *= 2.0 ** torch.randint(-14, 9, (rows, 1), device="cuda", generator=g)
        x[:, :cols // 3] *= 2.0 ** -9
        x[torch.rand(rows, device="cuda", generator=g) < 0.3] = 0.0
        x[5, 0], x[6, cols - 1], x[7, cols // 2] = float("nan"), float("inf"), -float("inf")
        x[9] = float("nan")
    elif kind == "tiny":
        x *= 2.0 ** -141
    elif kind == "huge":
        x[3] *= 2.0 ** 110
        x[rows - 2] *= 2.0 ** 120
    elif kind == "zero":
        x.zero_()
    return x.to(TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,rows,cols,layout", [
    ("normal", A.F16, 16384, 4096, A.MX_SCALES_TILED), ("normal", A.F16, 16400, 4099, A.MX_SCALES_TILED),
    ("outlier", A.F16, 16400, 4099, A.MX_SCALES_ROWS), ("outlier", A.BF16, 16403, 4096, A.MX_SCALES_TILED),
    ("few rows", A.F32, 8200, 4096, A.MX_SCALES_TILED), ("few rows", A.F16, 8400000, 5, A.MX_SCALES_ROWS),
    ("steep", A.F32, 8199, 4111, A.MX_SCALES_TILED), ("steep", A.BF16, 1680000, 40, A.MX_SCALES_TILED),
    ("steep", A.F16, 600, 120000, A.MX_SCALES_ROWS), ("tiny", A.F32, 8200, 4096, A.MX_SCALES_ROWS),
    ("huge", A.F32, 540, 65535, A.MX_SCALES_TILED), ("zero", A.F32, 8200, 4096, A.MX_SCALES_TILED)])
@pytest.mark.parametrize("offset", [0, 5])
def test_matrices_that_are_read_once(dev, kind, dtype, rows, cols, layout, offset):
    """Their factor is guessed and put right: the bytes are those of the right factor given from the start."""
    x = read_once_input(kind, dtype, rows, cols)
    top = float(x.float().abs().nan_to_num(nan=0.0, posinf=0.0).max())
    t = O.tensor_scale_of(top)
    runs = []
    for given in (None, t):
        h = Held(A.NVFP4, rows, cols, layout, t=given)
        if layout == A.MX_SCALES_ROWS:  # which may start anywhere
            h.m = mx.MxMatrix(A.NVFP4, rows, cols, h.codes.data_ptr(), h.scales.data_ptr() + offset, h.tensor.data_ptr(), ld=h.ld, layout=layout)
        values = torch.full((rows, cols), 7.0, dtype=x.dtype, device="cuda")
        dev.mx_quantize(x.data_ptr(), dtype, cols, h.m, values=values.data_ptr(), values_ld=cols, tensor_scale_given=given is not None)
        runs.append((h, values))
        if given is None:
            assert h.tensor.tolist() == [float(t), top]
    (found, values), (right, right_values) = runs
    assert torch.equal(found.scales, right.scales) and torch.equal(found.codes, right.codes)
    bits = torch.int32 if dtype == A.F32 else torch.int16
    assert torch.equal(values.view(bits), right_values.view(bits))
    some = torch.randint(0, rows, (40,)).unique().tolist() + [1, 5, rows - 1]
    q = O.quantize(x[some].cpu().double().numpy(), A.NVFP4, t=t)
    codes = found.codes[:rows * found.ld].view(rows, found.ld)[some].cpu().numpy()
    np.testing.assert_array_equal(codes[:, :found.pitch], O.pack(q["codes"]))
    if layout == A.MX_SCALES_ROWS:
        scales = found.scales[offset:offset + found.nscale].view(rows, -1)[some].cpu().numpy()
        np.testing.assert_array_equal(scales, q["scales"])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1.0, 0.37, 2.0 ** -9, 3e-30, 1e30])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_with_a_given_tensor_scale(dev, dtype, t):
    x = awkward(66, 200, dtype, 5)
    q = O.quantize(x.double().numpy(), A.NVFP4, t=np.float32(t))
    h = Held(A.NVFP4, 66, 200, A.MX_SCALES_TILED, t=t)
    src = put(x, 0)
    dev.mx_quantize(src.data_ptr(), dtype, src.stride(0), h.m, tensor_scale_given=True)
    h.check(q)
    assert h.tensor.tolist() == [float(np.float32(t)), -1.0]  # read, not written


def steps_from(x, steps):
    """32-bit numbers so many units in the last place from x."""
    return (np.asarray(x, np.float32)[..., None].view(np.int32) + np.asarray(steps, np.int32)).view(np.float32)


def next_to_borders(t, scales):
    """Rows of blocks for the tensor scale t: each block's largest element gives it one of `scales`, its others lie next
    to the borders between the codes of 4 bits."""
    e4m3 = O.e4m3_values()[scales].astype(np.float32)
    d = e4m3 * np.float32(t)  # rounded to 32 bits, as the definition says
    v = steps_from(d[:, None] * np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32), range(-3, 4)).reshape(len(d), 49)
    x = np.zeros((len(d), 64), np.float32)
    x[:, ::16] = (6 * d)[:, None]
    x[:, [i for i in range(64) if i % 16][:49]] = v * np.where(np.arange(49) % 3 == 1, -1, 1).astype(np.float32)
    return x


def next_to_scales(t):
    """One block a row, whose largest element lies next to a border between two of e4m3's numbers."""
    values = O.e4m3_values()[:127]
    top = steps_from((np.float32(6) * np.float32(t)) * ((values[1:] + values[:-1]) / 2).astype(np.float32), range(-3, 4)).reshape(-1)
    x = np.zeros((len(top), 16), np.float32)
    x[:, 5] = top
    return x


def check_quotients(dev, x, t):
    h = Held(A.NVFP4, x.shape[0], x.shape[1], A.MX_SCALES_ROWS, t=t)
    src = torch.from_numpy(x).cuda()
    dev.mx_quantize(src.data_ptr(), A.F32, x.shape[1], h.m, tensor_scale_given=True)
    h.check(O.quantize(x, A.NVFP4, t=np.float32(t)))


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [0, -30, 21, -100, 90])
@pytest.mark.parametrize("eighths", range(8, 17))
def test_quotients_of_the_divisors_that_could_be_misrounded(dev, eighths, exponent):
    """Full-width divisors for which a rounded quotient may fall on a border although the quotient does not: those within
    some units in the last place of a multiple of 1/8.  Every one of them, against correctly rounded quotients."""
    near = steps_from(np.float32(eighths / 8), range(-64, 65))
    for d in near:
        t = float(d) * 2.0 ** exponent
        check_quotients(dev, next_to_borders(t, np.array([56, 48, 64])), t)  # scales of 1, 0.5 and 2: d is t
    for six in near:
        for t in steps_from(six / np.float32(6) * np.float32(2.0 ** exponent), (-1, 0, 1)):
            if np.float32(6) * t == np.float32(float(six) * 2.0 ** exponent):
                check_quotients(dev, next_to_scales(t), float(t))
                break


@pytest.mark.gpu
def test_quotients_of_random_divisors(dev):
    rng = np.random.default_rng(21)
    for _ in range(150):
        t = float(np.float32(rng.uniform(1, 2) * 2.0 ** rng.integers(-30, 20)))
        check_quotients(dev, next_to_borders(t, np.arange(1, 127)), t)
        check_quotients(dev, next_to_scales(t), t)


def test_borders_of_the_codes_and_their_neighbours():
    """The inputs of the tests above reach both sides of every border, and the border itself."""
    t = np.float32(1.5)
    q = O.quantize(next_to_borders(t, np.array([56])), A.NVFP4, t=t)["codes"][0] & 7
    assert set(q) == set(range(8))
    s = O.quantize(next_to_scales(t), A.NVFP4, t=t)["scales"]
    assert set(s.reshape(-1)) == set(range(127))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_extreme_magnitudes(dev, fmt):
    """Every exponent of 32 bits, so that scales reach both ends of their range."""
    rows = 254
    e = np.arange(rows)[:, None] - 126.0
    x = (np.random.default_rng(2).uniform(-1.99, 1.99, (rows, 64)) * 2.0 ** e).astype(np.float32)
    for part in (x, x[:100], x[100:150]):
        h = Held(fmt, len(part), 64, A.MX_SCALES_ROWS)
        src = torch.from_numpy(part.copy()).cuda()
        dev.mx_quantize(src.data_ptr(), A.F32, 64, h.m)
        h.check(O.quantize(part, fmt))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan"), float("inf")])
def test_given_scales_that_are_no_scales(dev, bad):
    h = Held(A.NVFP4, 3, 32, A.MX_SCALES_ROWS, t=bad)
    src = torch.ones(3, 32, device="cuda")
    dev.mx_quantize(src.data_ptr(), A.F32, 32, h.m, tensor_scale_given=True)
    assert (h.scales[:h.nscale] == 127).all() and (h.codes[:3 * 16] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", FORMATS)
def test_dequantize(dev, fmt, dtype, rows, cols):
    rng = np.random.default_rng(rows + cols)
    blocks = -(-cols // O.BLOCK[fmt])
    # every scale byte that may be there, NaN among them
    q = dict(codes=rng.integers(0, 16, (rows, cols)).astype(np.uint8),
             scales=rng.integers(0, 256 if fmt == A.MXFP4 else 128, (rows, blocks)).astype(np.uint8), t=np.float32(0.3))
    want = O.values_of(q["codes"], q["scales"], fmt, q["t"])
    for layout, pad, extra in ((A.MX_SCALES_ROWS, 0, 16), (A.MX_SCALES_TILED, 8, 0), (A.MX_SCALES_TILED, 1, 0)):
        h = Held(fmt, rows, cols, layout, extra).load(q)
        out = torch.full((rows, cols + pad), 7.0, dtype=TYPES[dtype], device="cuda")
        dev.mx_dequantize(h.m, out.data_ptr(), dtype, out.stride(0))
        got = out[:, :cols].cpu()
        # scale * t is rounded to 32 bits, code times that again, then the type rounds: with |w| the exact value,
        # (2 * 2^-24 + eps / 2) |w| and a little for their product; half of the smallest step below the normal range
        info = torch.finfo(TYPES[dtype])
        with np.errstate(over="ignore"):
            bound = np.abs(want) * (2 * 2.0 ** -24 + info.eps / 2) * 1.001 + info.smallest_normal * info.eps / 2 * 1.001
        g = got.double().numpy()
        nan = np.isnan(want)
        assert (np.isnan(g) == nan).all()
        over = np.abs(want) >= info.max * (1 + info.eps / 4)  # rounds to infinity
        border = (np.abs(want) > info.max) & ~over
        ok = np.abs(np.where(nan | over | border | np.isinf(g), 0, g - want)) <= bound
        assert ok[~nan].all()
        assert np.isinf(g[over & ~nan]).all() and not np.isinf(g[~over & ~border & ~nan]).any()
        assert (out[:, cols:] == 7.0).all()


@pytest.mark.gpu
def test_empty_matrices(dev):
    for rows, cols in ((0, 5), (5, 0), (0, 0)):
        for fmt in FORMATS:
            h = Held(fmt, rows, cols, A.MX_SCALES_TILED)
            src = torch.ones(8, 8, device="cuda")
            dev.mx_quantize(src.data_ptr(), A.F32, 8, h.m)
            dev.mx_dequantize(h.m, src.data_ptr(), A.F32, 8)
            assert (h.codes == CANARY).all() and (h.scales == CANARY).all() and (src == 1).all()
            if fmt == A.NVFP4:
                assert h.tensor.tolist() == [1.0, 0.0]


# --------------------------------------------------------------------------- product
@pytest.mark.parametrize("change,said", [
    (dict(), "null context"), (dict(dtype=A.I8), "element type"), (dict(ld=63), "fewer elements"), (dict(out=None), "output: null"),
    (dict(out=0x10000), "overlaps codes"), (dict(out=0x51000), "overlaps scales"), (dict(a=dict(fmt=A.MXFP4)), "different formats"),
    (dict(a=dict(cols=96, ld=48)), "different numbers"), (dict(a=dict(layout=A.MX_SCALES_ROWS)), "tiled scales"),
    (dict(b=dict(layout=A.MX_SCALES_ROWS)), "tiled scales"), (dict(b=dict(tensor_scale=None)), "needs a tensor scale"),
    (dict(a=dict(codes=0x10001)), "16-byte"), (dict(a=dict(rows=1, ld=1 << 41), ld=1 << 42, out=1 << 50), "too large for a product"), (dict(a=dict(ld=24)), "multiple of 16"),
])
def test_matmul_refusals(change, said):
    a = matrix(**dict(dict(ld=32), **change.get("a", {})))
    b = matrix(**dict(dict(ld=32, codes=0x50000, scales=0x51000, tensor_scale=0x52000), **change.get("b", {})))
    args = dict(dict(out=0x100000, dtype=A.F32, ld=64), **{k: v for k, v in change.items() if k not in "ab"})
    assert said in refused("b200c_mx_matmul", C.byref(a.c), C.byref(b.c), args["out"], args["dtype"], args["ld"])
    assert "null descriptor" in refused("b200c_mx_matmul", None, C.byref(b.c), args["out"], args["dtype"], args["ld"])


def random_held(fmt, rows, cols, seed, spread=4, extra_ld=0):
    """A matrix of random codes and scales in the product's layout: scales over 2^(2 * spread)."""
    rng = np.random.default_rng(seed)
    blocks = -(-cols // O.BLOCK[fmt])
    mid = 127 if fmt == A.MXFP4 else 56
    step = 1 if fmt == A.MXFP4 else 8
    scales = rng.integers(mid - spread * step, mid + spread * step + 1, (rows, blocks)).astype(np.uint8)
    q = dict(codes=rng.integers(0, 16, (rows, cols)).astype(np.uint8), scales=scales, t=np.float32(2.0 ** -rng.integers(0, 9)))
    return Held(fmt, rows, cols, A.MX_SCALES_TILED, extra_ld).load(q), O.values_of(q["codes"], q["scales"], fmt, q["t"])


def check_product(got, va, vb, dtype):
    want = va @ vb.T
    size = np.abs(va) @ np.abs(vb).T
    # products are exact; a step of 64 adds to the 32-bit sum with at most one unit in the last place lost, and the
    # sums' scale once more; then the type rounds, half a step of its subnormal range at least
    steps = -(-va.shape[1] // 64) + 2
    info = torch.finfo(TYPES[dtype])
    bound = steps * 2.0 ** -23 * size + np.abs(want) * info.eps / 2 * (1 + 2.0 ** -10) + info.smallest_normal * info.eps / 2
    over = np.abs(want) > info.max
    assert not np.isnan(got).any()
    far = np.where(over, 0, np.abs(got - want)) - bound
    assert (far <= 0).all(), (far.max(), np.unravel_index(far.argmax(), far.shape))


PRODUCTS = [(1, 1, 1), (1, 128, 32), (3, 5, 16), (16, 130, 100), (17, 300, 257), (64, 64, 64), (65, 1000, 515), (128, 129, 300),
            (129, 128, 1003), (200, 300, 4100), (300, 20, 777), (257, 513, 2048), (1, 1000, 11008), (130, 1, 96),
            # from here on the two-CTA form: a stage and less, several tiles per pair, ragged edges
            (1537, 1700, 40), (1537, 1700, 1003), (257, 4900, 515), (2600, 2700, 300), (4864, 257, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul(dev, fmt, m, n, k):
    a, va = random_held(fmt, m, k, m + k, extra_ld=16 if n % 2 else 0)
    b, vb = random_held(fmt, n, k, n + 3 * k)
    for dtype, pad in ((A.F32, 0), (A.BF16, 8), (A.F16, 3)):
        out = torch.full((m, n + pad), 7.0, dtype=TYPES[dtype], device="cuda")
        dev.mx_matmul(a.m, b.m, out.data_ptr(), dtype, out.stride(0))
        dev.synchronize()
        got = out.double().cpu().numpy()
        check_product(got[:, :n], va, vb, dtype)
        assert (got[:, n:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1507, 1789), (1600, 1785), (1601, 1792), (1537, 1704), (1600, 1808), (1537, 2057), (4900, 257), (129, 5001), (300, 1003),
                                 (3, 129), (40, 700)])
@pytest.mark.parametrize("k", [40, 700])
@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_writes_its_columns_alone(dev, fmt, m, n, k):
    """Results inside a wider matrix whose rows are aligned: the columns behind the last, in its 16-byte line and
    further, and the row behind the last stay as they were."""
    (a, va), (b, vb) = random_held(fmt, m, k, m), random_held(fmt, n, k, n)
    for dtype in TYPES:
        line = 128 // torch.finfo(TYPES[dtype]).bits
        for ld in (-(-n // line) * line, -(-n // line) * line + line):
            out = torch.full((m * ld + 3 * line,), 7.0, dtype=TYPES[dtype], device="cuda")
            dev.mx_matmul(a.m, b.m, out.data_ptr(), dtype, ld)
            body, behind = out[:m * ld].view(m, ld), out[m * ld:]
            check_product(body[:, :n].double().cpu().numpy(), va, vb, dtype)
            assert (body[:, n:] == 7.0).all() and (behind == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(16, 256, 1024), (300, 700, 2048), (1600, 1800, 2048)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_is_exact_where_sums_are(dev, fmt, m, n, k):
    """Scales of one: every product is a multiple of 1/4 below 36, so sums of up to 2^17 of them fit 24 bits."""
    rng = np.random.default_rng(k)
    one = 127 if fmt == A.MXFP4 else 56
    sides = []
    for rows in (m, n):
        q = dict(codes=rng.integers(0, 16, (rows, k)).astype(np.uint8),
                 scales=np.full((rows, k // O.BLOCK[fmt]), one, np.uint8), t=np.float32(1))
        sides.append((Held(fmt, rows, k, A.MX_SCALES_TILED).load(q), O.decode(q["codes"])))
    (a, va), (b, vb) = sides
    out = torch.empty(m, n, device="cuda")
    dev.mx_matmul(a.m, b.m, out.data_ptr(), A.F32, n)
    np.testing.assert_array_equal(out.double().cpu().numpy(), va @ vb.T)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(5, 40, 64), (5, 300, 2048), (129, 200, 512), (1600, 1800, 128), (1537, 1701, 300)])
@pytest.mark.parametrize("ta,tb", [(2.0 ** -75, 2.0 ** -75), (2.0 ** -75 * 1.37, 2.0 ** -80 * 1.91), (2.0 ** 65, 2.0 ** 65), (2.0 ** 70 * 1.7, 2.0 ** 59),
                                   (2.0 ** -100, 2.0 ** 100), (3e38, 2e-38), (2.0 ** -149, 2.0 ** 20), (2.0 ** -140 * 3, 2.0 ** 10 * 1.3),
                                   (2.0 ** -126, 2.0 ** -126), (3e38, 3e38), (2.0 ** -149, 2.0 ** -149)])
def test_matmul_over_the_range_of_the_tensor_scales(dev, m, n, k, ta, tb):
    """Their product may leave 32 bits where the results do not; rows of zeros stay zeros."""
    (a, va), (b, vb) = random_held(A.NVFP4, m, k, m + 5, spread=6), random_held(A.NVFP4, n, k, n + 6, spread=6)
    for h, v, t in ((a, va, ta), (b, vb, tb)):
        v *= float(np.float32(t)) / float(h.tensor[0])
        h.tensor[0] = float(np.float32(t))
        v[1] = 0
        h.codes[:h.rows * h.ld].view(h.rows, h.ld)[1] = 0
    # what is above the largest number by more than half a step, and by what a sum may be off (see check_product)
    above = np.abs(va @ vb.T) - (-(-k // 64) + 2) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)
    for dtype, pad in ((A.F32, 0), (A.BF16, 8), (A.F16, 3)):
        out = torch.full((m, n + pad), 7.0, dtype=TYPES[dtype], device="cuda")
        dev.mx_matmul(a.m, b.m, out.data_ptr(), dtype, out.stride(0))
        got = out[:, :n].double().cpu().numpy()
        check_product(got, va, vb, dtype)
        assert (got[1] == 0).all() and (got[:, 1] == 0).all()
        info = torch.finfo(TYPES[dtype])
        assert np.isinf(got[above > info.max * (1 + info.eps)]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(20, 150, 200), (1700, 1601, 200)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_keeps_nan_to_its_rows(dev, fmt, m, n, k):
    """A NaN scale in one row of each side; the scales that fill up the tiles are NaN too, and must not matter."""
    a, va = random_held(fmt, m, k, 1)
    b, vb = random_held(fmt, n, k, 2)
    nan = 255 if fmt == A.MXFP4 else 127
    want = va @ vb.T
    for h, rows in ((a, m), (b, n)):
        mark = np.zeros((-(-rows // 128) * 128, -(-k // O.BLOCK[fmt])), np.uint8)
        mark[rows:] = 1  # rows behind the last
        mark[7, 3] = 1
        laid = torch.from_numpy(O.lay(mark, 1)).cuda().bool()
        h.scales[:h.nscale][laid] = nan
    out = torch.empty(m, n, device="cuda")
    dev.mx_matmul(a.m, b.m, out.data_ptr(), A.F32, n)
    got = out.double().cpu().numpy()
    bad = np.zeros((m, n), bool)
    bad[7], bad[:, 7] = True, True
    assert np.isnan(got[bad]).all()
    assert np.isfinite(got[~bad]).all() and np.allclose(got[~bad], want[~bad], rtol=1e-4, atol=1e-4 * np.abs(want).max())


@pytest.mark.gpu
def test_matmul_of_nothing(dev):
    for fmt in FORMATS:
        a, b = Held(fmt, 3, 0, A.MX_SCALES_TILED), Held(fmt, 5, 0, A.MX_SCALES_TILED)
        out = torch.full((3, 6), 7.0, device="cuda")
        dev.mx_matmul(a.m, b.m, out.data_ptr(), A.F32, 6)
        assert (out[:, :5] == 0).all() and (out[:, 5] == 7).all()
        e, f = Held(fmt, 0, 64, A.MX_SCALES_TILED), Held(fmt, 5, 64, A.MX_SCALES_TILED)
        dev.mx_matmul(e.m, f.m, out.data_ptr(), A.F32, 6)
        dev.mx_matmul(f.m, e.m, out.data_ptr(), A.F32, 6)
        assert (out[:, 5] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_then_multiply(dev, fmt):
    """A linear layer as a program runs it: weights once, activations and the product every time, also captured."""
    m, n, k = 5, 200, 300
    rng = np.random.default_rng(9)
    w = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32)).half()
    qw = O.quantize(w.double().numpy(), fmt)
    hw = Held(fmt, n, k, A.MX_SCALES_TILED)
    dw = w.cuda()
    dev.mx_quantize(dw.data_ptr(), A.F16, k, hw.m)
    hx = Held(fmt, m, k, A.MX_SCALES_TILED)
    dx = torch.zeros(m, k, dtype=torch.half, device="cuda")
    out = torch.empty(m, n, dtype=torch.half, device="cuda")

    def step():
        dev.mx_quantize(dx.data_ptr(), A.F16, k, hx.m)
        dev.mx_matmul(hx.m, hw.m, out.data_ptr(), A.F16, n)

    def check(x):
        qx = O.quantize(x.double().numpy(), fmt)
        check_product(out.double().cpu().numpy(), qx["values"], qw["values"], A.F16)

    xs = [torch.from_numpy(rng.standard_normal((m, k)) * s).half() for s in (1.0, 30.0)]
    dx.copy_(xs[0])
    step()
    check(xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dev.set_stream(torch.cuda.current_stream().cuda_stream)
        step()
    dev.set_stream(torch.cuda.current_stream().cuda_stream)
    for x in (xs[1], xs[0]):
        dx.copy_(x)
        graph.replay()
        check(x)


# --------------------------------------------------------------------------- as programs use them together
@pytest.mark.gpu
def test_rows_far_apart(dev):
    """Offsets beyond 2^31 elements and 2^32 bytes: three rows with a gigabyte and more between them."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    rows, cols, far = 3, 70, (1 << 30) + 24
    x = awkward(rows, cols, A.F16, 1, special=False)
    for fmt in FORMATS:
        q = O.quantize(x.double().numpy(), fmt)
        src = torch.empty(2 * far + cols, dtype=torch.half, device="cuda")
        view = src.as_strided((rows, cols), (far, 1))
        view.copy_(x.cuda())
        ld = (1 << 31) + 32
        codes = torch.empty(2 * ld + 48, dtype=torch.uint8, device="cuda")
        scales = torch.empty(mx.sizes(fmt, rows, cols)[2], dtype=torch.uint8, device="cuda")
        tensor = torch.zeros(2, device="cuda")
        m = mx.MxMatrix(fmt, rows, cols, codes.data_ptr(), scales.data_ptr(), tensor.data_ptr(), ld=ld)
        dev.mx_quantize(src.data_ptr(), A.F16, far, m)
        np.testing.assert_array_equal(codes.as_strided((rows, 48), (ld, 1)).cpu().numpy(), O.pack(q["codes"]))
        src.as_strided((rows, cols), (far, 1)).zero_()
        dev.mx_dequantize(m, src.data_ptr(), A.F16, far)
        np.testing.assert_array_equal(view.cpu().numpy(), q["values"].astype(np.float32).astype(np.float16))
        out = src.as_strided((rows, rows), (far, 1))
        dev.mx_matmul(m, m, src.data_ptr(), A.F16, far)
        check_product(out.double().cpu().numpy(), q["values"], q["values"], A.F16)
        del src, view, out, codes


@pytest.mark.gpu
def test_two_contexts_on_two_streams_from_two_threads(dev):
    """Each with its own matrices; the results are those of one after the other."""
    import threading
    from npu_plugin_b200.const import CudaBackend
    shapes = [(40, 3000, 2000), (1600, 1900, 520)]
    made = []
    for i, (m, n, k) in enumerate(shapes):
        a, _ = random_held(A.NVFP4, m, k, i)
        b, _ = random_held(A.NVFP4, n, k, i + 7)
        want = torch.empty(m, n, device="cuda")
        dev.mx_matmul(a.m, b.m, want.data_ptr(), A.F32, n)
        made.append((a, b, want, torch.empty(m, n, device="cuda")))
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            backend = CudaBackend(0)
            a, b, _, out = made[i]
            for _ in range(50):
                backend.mx_matmul(a.m, b.m, out.data_ptr(), A.F32, out.shape[1])
            backend.synchronize()
            backend.close()
        except Exception as e:
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for _, _, want, out in made:
        assert torch.equal(want, out)


@pytest.mark.gpu
def test_two_graphs_in_turn_and_every_result_the_same_bytes(dev):
    """Two captured layers that share their weights, replayed in turn, against eager runs."""
    n, k = 700, 1100
    w, _ = random_held(A.MXFP4, n, k, 3)
    cases = []
    for m in (3, 150):
        g = torch.Generator().manual_seed(m)
        x = torch.randn(m, k, generator=g).bfloat16().cuda()
        h = Held(A.MXFP4, m, k, A.MX_SCALES_TILED)
        out = torch.zeros(m, n, device="cuda")

        def step(x=x, h=h, out=out):
            dev.mx_quantize(x.data_ptr(), A.BF16, k, h.m)
            dev.mx_matmul(h.m, w.m, out.data_ptr(), A.F32, n)
        step()
        torch.cuda.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dev.set_stream(torch.cuda.current_stream().cuda_stream)
            step()
        dev.set_stream(torch.cuda.current_stream().cuda_stream)
        cases.append((graph, out, want, x, h))  # the graph reads x and writes h: they have to live as long
    for _ in range(20):
        for graph, out, *_ in cases:
            out.zero_()
            graph.replay()
        for _, out, want, *_ in cases:
            assert torch.equal(out, want)


@pytest.mark.gpu
def test_first_use_inside_a_capture():
    """A process whose very first calls are captured."""
    import os
    import subprocess
    import sys
    code = """
import torch
from npu_plugin_b200 import _cabi as A, const, mx
b = const.CudaBackend(0)
x = torch.randn(300, 640, device="cuda").half()
out = torch.zeros(300, 300, device="cuda")
ld, nc, ns = mx.sizes(A.NVFP4, 300, 640)
codes, scales, t = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (nc, ns, 8))
m = mx.MxMatrix(A.NVFP4, 300, 640, codes.data_ptr(), scales.data_ptr(), t.data_ptr())
back = torch.empty_like(x)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    b.mx_quantize(x.data_ptr(), A.F16, 640, m)
    b.mx_dequantize(m, back.data_ptr(), A.F16, 640)
    b.mx_matmul(m, m, out.data_ptr(), A.F32, 300)
g.replay()
torch.cuda.synchronize()
v = back.double()
assert (out.double() - v @ v.t()).abs().max() < 1e-3 * 640
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
