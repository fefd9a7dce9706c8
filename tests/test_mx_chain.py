"""Block-scaled 4-bit floats as transformations of a constant: QuantizeMx and DequantizeMx in chains, in batched folds,
through the constant-folding pass, and the chain builder that decides whether a layer's weights may be held so."""
import gc
import time

import numpy as np
import pytest

import mx_oracle as O
from npu_plugin_b200 import _cabi as A
from npu_plugin_b200 import chains
from npu_plugin_b200.blob import ConstantDecl, ShardFolder
from npu_plugin_b200.cache import (ConstantFoldingCacheManager, initBackgroundConstantFoldingThreads,
                                   stopBackgroundConstantFoldingThreads)
from npu_plugin_b200.const import (ConstError, Content, ContentAttr, DeclareOp, DimsOrder, NDType, ResidentContent, Transform,
                                   Unsupported, constant_folding_pass)
from test_abi_and_host import HostOnly

FORMATS = [A.MXFP4, A.NVFP4]
Q = lambda fmt, **kw: Transform(A.X_QUANTIZE_MX, i0=fmt, **kw)
D = lambda fmt, elem=A.F16, **kw: Transform(A.X_DEQUANTIZE_MX, i0=fmt, elem=elem, **kw)


# --------------------------------------------------------------------------- types and refusals, without a device
def test_types():
    host = HostOnly()
    t = host.infer_type(NDType((8, 64), A.F16), [Q(A.NVFP4)])
    assert (t.shape, t.dtype, t.getTotalAllocSize()) == ((8, 64), A.F4E2M1, 256)
    t = host.infer_type(NDType((8, 16, 3, 64), A.F32, DimsOrder.NHWC), [Transform(A.X_PAD_WITH_ZERO, a=(0,) * 4, b=(0, 16, 0, 0)), Q(A.MXFP4)])
    assert (t.shape, t.dtype, tuple(t.order)) == ((8, 32, 3, 64), A.F4E2M1, (0, 2, 3, 1))
    t = host.infer_type(NDType((8, 64), A.F16), [Q(A.NVFP4), Transform(A.X_SWIZZLE_CONSTANT, i0=5, i1=3)])
    assert (t.shape, t.dtype) == ((512, 1, 1, 1), A.UI8)
    assert host.infer_type(NDType((8, 64), A.F16), [Q(A.NVFP4), D(A.NVFP4, A.F32)]).dtype == A.F32
    assert host.insert_position([A.X_QUANTIZE_MX], A.X_DEQUANTIZE_MX) == 1


@pytest.mark.parametrize("base,chain,error,said", [
    (NDType((8, 40), A.F16), [Q(A.NVFP4)], ConstError, "multiple of 32"),
    (NDType((8, 64), A.UI8), [Q(A.NVFP4)], ConstError, "expects an f16"),
    (NDType((8, 64), A.F64), [Q(A.MXFP4)], ConstError, "expects an f16"),
    (NDType((8, 64), A.F16), [Q(7)], ValueError, "unknown block-scaled format"),
    (NDType((8, 64), A.F16), [Q(A.MXFP4, f=1.0)], ValueError, "nvfp4's alone"),
    (NDType((8, 64), A.F16), [Q(A.NVFP4, f=-1.0)], ValueError, "positive"),
    (NDType((8, 64), A.F16), [Q(A.NVFP4, f=1e-60)], ValueError, "positive"),
    (NDType((8, 64), A.F16), [Q(A.NVFP4, f=float("nan"))], ValueError, "positive"),
    (NDType((8, 64), A.F16), [D(A.NVFP4)], ConstError, "expects a tensor of 4-bit floats"),
    (NDType((8, 64), A.F4E2M1), [D(A.NVFP4, A.F64)], ValueError, "needs the element type"),
    (NDType((8, 16), A.F4E2M1), [D(A.NVFP4)], ConstError, "multiple of 32"),
    (NDType((8, 64), A.F16), [Transform(A.X_CONVERT_ELEM_TYPE, elem=A.F4E2M1)], ValueError, "come from QuantizeMx"),
    (NDType((8, 64), A.F4E2M1), [Transform(A.X_CONVERT_ELEM_TYPE, elem=A.F16)], ValueError, "go through DequantizeMx"),
    (NDType((), A.F16), [Q(A.NVFP4)], ConstError, "multiple of 32"),
])
def test_refused_chains(base, chain, error, said):
    with pytest.raises(error, match=said):
        HostOnly().infer_type(base, chain)


def test_scales_on_the_host_are_refused_where_the_fold_runs_on_the_device():
    class Backend(HostOnly):
        ctx = None
    d = ConstantDecl("w", NDType((8, 64), A.F16), [Q(A.NVFP4, side0=np.zeros((8, 4), np.uint8))], 1024)
    with pytest.raises(ValueError, match="have to lie there"):
        ShardFolder(Backend(), [d])


def test_wrong_numbers_of_scales_are_refused():
    attr = ContentAttr(np.zeros(256, np.uint8), NDType((8, 64), A.F4E2M1), False, [], HostOnly())
    with pytest.raises(ConstError, match="31 scales for 32 blocks"):
        attr.dequantizeMx(A.NVFP4, A.F16, scales=np.zeros(31, np.uint8), tensorScale=[1.0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_have_the_shape_of_what_is_quantised(fmt):
    """Swizzling stays behind, whichever was asked for first."""
    host = HostOnly()
    w = ContentAttr.get(np.zeros((8, 256), np.float16), is_splat=False, backend=host)
    for q in (w.quantizeMx(fmt), w.quantizeMx(fmt).swizzleConstant(5, 3), w.swizzleConstant(5, 3).quantizeMx(fmt)):
        assert q.mxScales.shape == (8, 256 // O.BLOCK[fmt])
    stored = ContentAttr.get(np.zeros(1024, np.uint8), NDType((8, 256), A.F4E2M1), False, host)
    scales = np.zeros((8, 256 // O.BLOCK[fmt]), np.uint8)
    back = stored.swizzleConstant(5, 3).dequantizeMx(fmt, A.F16, scales, [1.0] if fmt == A.NVFP4 else None)
    assert [t.kind for t in back.getTransformations()] == [A.X_DEQUANTIZE_MX, A.X_SWIZZLE_CONSTANT]
    s = w.swizzleConstant(5, 3).quantizeSynth(A.QSYNTH_SYM_I8)
    assert s.sideScales.shape == s.sideZeroPoints.shape == (8,)


def test_two_transformations_with_their_own_scales_are_not_one():
    s = np.zeros((8, 2), np.uint8)
    assert Q(A.MXFP4, side0=s) == Q(A.MXFP4, side0=s)
    assert Q(A.MXFP4, side0=s) != Q(A.MXFP4, side0=s.copy())


# --------------------------------------------------------------------------- background folding
class FakeDevice(HostOnly):
    """Folds lists of one QuantizeMx and one DequantizeMx with the oracle, into host memory."""

    def __init__(self):
        super().__init__()
        self.folds = 0

    def _run(self, base_type, data, transforms):
        self.folds += 1
        q = None
        for t in transforms:
            rows, cols = base_type.shape
            if t.kind == A.X_QUANTIZE_MX:
                q = O.quantize(data.astype(np.float64), t.i0, t=t.f or None)
                t.side0[:] = q["scales"]
                if t.i0 == A.NVFP4:
                    t.side1[:] = q["t"], q["top"]
                out = O.pack(q["codes"]).reshape(-1)
            else:
                packed = data.reshape(rows, -1) if q is None else O.pack(q["codes"])
                codes = np.stack([packed & 15, packed >> 4], 2).reshape(rows, -1)[:, :cols]
                scales = q["scales"] if t.side0 is None else t.side0.reshape(rows, -1)
                factor = q["t"] if t.side0 is None else None if t.side1 is None else t.side1[0]
                out = O.values_of(codes, scales, t.i0, factor).astype(np.float32).reshape(-1)
        return out.view(np.uint8)

    def fold(self, base_type, data, is_splat, transforms):
        out = self._run(base_type, data, transforms)
        return Content(self.infer_type(base_type, transforms), out, out.size)

    def fold_resident(self, base_type, data, is_splat, transforms):
        out = self._run(base_type, data, transforms)
        return ResidentContent(self, self.infer_type(base_type, transforms), out, out.size, out.size)

    def resident_to_host(self, rc):
        return rc.buf

    def free_resident(self, rc):
        rc.buf = None


@pytest.fixture(params=["fake", pytest.param("b200", marks=pytest.mark.gpu)])
def folding_ahead(request):
    """A context whose attributes are folded by two threads as they are built."""
    if request.param == "fake":
        ctx = FakeDevice()
    else:
        from npu_plugin_b200.const import CudaBackend
        ctx = CudaBackend(0)
    threads = initBackgroundConstantFoldingThreads(ctx, 2)
    yield ctx
    stopBackgroundConstantFoldingThreads(ctx, threads)


@pytest.mark.parametrize("fmt", FORMATS)
def test_each_attribute_receives_its_scales_from_the_cache(folding_ahead, fmt):
    """Attributes of one base that are built, folded and dropped: an address that comes back is another array."""
    w = np.random.default_rng(11).normal(0, 1, (6, 64)).astype(np.float32)
    want = O.quantize(w.astype(np.float64), fmt)
    base = ContentAttr.get(w, backend=folding_ahead)
    for _ in range(20):
        q = base.quantizeMx(fmt)
        np.testing.assert_array_equal(q.fold().copyTo(), O.pack(want["codes"]).reshape(-1))
        np.testing.assert_array_equal(q.mxScales, want["scales"])
        if fmt == A.NVFP4:
            assert q.mxTensorScale.tolist() == [want["t"], want["top"]]
        back = q.dequantizeMx(fmt, A.F32)
        q.mxScales[:] = 0
        np.testing.assert_array_equal(back.fold().getValues().reshape(w.shape), want["values"].astype(np.float32))
        np.testing.assert_array_equal(q.mxScales, want["scales"])  # those of one transformation: written again
        del q, back
        gc.collect()


@pytest.mark.parametrize("fmt", FORMATS)
def test_each_attribute_is_read_with_its_own_scales(folding_ahead, fmt):
    rng = np.random.default_rng(12)
    codes = rng.integers(0, 16, (6, 64)).astype(np.uint8)
    base = ContentAttr.get(O.pack(codes).reshape(-1), NDType((6, 64), A.F4E2M1), is_splat=False, backend=folding_ahead)
    blocks = (6, 64 // O.BLOCK[fmt])
    scales, factor = np.zeros(blocks, np.uint8), np.zeros(2, np.float32)
    for i in range(20):
        if i % 2:  # the same arrays with other numbers in them, or others that may come to lie where the last ones did
            scales, factor = np.empty(blocks, np.uint8), np.empty(2, np.float32)
        scales[:], factor[0] = rng.integers(40, 80, blocks), rng.uniform(0.5, 2.0)
        want = O.values_of(codes, scales, fmt, factor[0])
        a = base.dequantizeMx(fmt, A.F32, scales, factor if fmt == A.NVFP4 else None)
        scales[:], factor[0] = 0, 0  # what was given counts
        # scale * factor is rounded to 32 bits, code times that again: half a unit of 2^-23 each, and their product
        np.testing.assert_allclose(a.fold().getValues().reshape(6, 64).astype(np.float64), want, rtol=2 * 2.0 ** -24 * 1.001, atol=0)
        del a
        gc.collect()


def test_bases_at_one_address_are_not_one(folding_ahead):
    for i in range(20):
        q = ContentAttr.get(np.full((1, 32), i + 1.0, np.float32), is_splat=False, backend=folding_ahead).quantizeMx(A.MXFP4)
        q.fold()
        np.testing.assert_array_equal(q.mxScales, O.quantize(np.full((1, 32), i + 1.0), A.MXFP4)["scales"])
        del q
        gc.collect()


def test_one_fold_answers_all_that_ask_for_the_same():
    ctx = FakeDevice()
    w = np.random.default_rng(13).normal(0, 1, (6, 64)).astype(np.float32)
    base = ContentAttr.get(w, backend=ctx)
    threads = initBackgroundConstantFoldingThreads(ctx, 1)
    attrs = [base.quantizeMx(A.MXFP4) for _ in range(5)]
    while not ConstantFoldingCacheManager.getInstance().get(ctx)._requests.empty():
        time.sleep(0.01)
    for a in attrs:
        a.fold()
        assert (a.mxScales == attrs[0].mxScales).all() and (a.mxScales != 0).all()
    assert ctx.folds == 1 and attrs[0] is not attrs[1] and attrs[0].mxScales is not attrs[1].mxScales
    stopBackgroundConstantFoldingThreads(ctx, threads)


def test_the_callers_memory_is_never_read_or_written_ahead():
    """Side arrays given as addresses: nobody but the caller knows what lies there, and when."""
    ctx = FakeDevice()
    threads = initBackgroundConstantFoldingThreads(ctx, 1)
    base = ContentAttr.get(np.zeros((2, 32), np.float32), is_splat=False, backend=ctx)
    a = base.addTransformation(Q(A.MXFP4, side0=0x1000))
    b = a.addTransformation(D(A.MXFP4))
    stopBackgroundConstantFoldingThreads(ctx, threads)
    assert ctx.folds == 0 and not a.isCacheable() and not b.isCacheable() and base.quantizeMx(A.MXFP4).isCacheable()


# --------------------------------------------------------------------------- on the device
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_conv_weight_chain(gpu, oracle, fmt):
    """OIYX f32 weights -> OYXI -> input channels padded to a multiple of 32 -> 4 bits, also swizzled and read back."""
    w = np.random.default_rng(3).normal(0, 0.05, (24, 40, 3, 3)).astype(np.float32)
    a = ContentAttr.get(w, NDType(w.shape, A.F32), backend=gpu).reorder(DimsOrder.OYXI).padWithZero((0,) * 4, (0, 24, 0, 0))
    q = a.quantizeMx(fmt)
    x = np.pad(w.transpose(0, 2, 3, 1), ((0, 0),) * 3 + ((0, 24),)).reshape(-1, 64)
    want = O.quantize(x, fmt)
    c = q.fold()
    assert c.getType().dtype == A.F4E2M1 and c.getType().shape == (24, 64, 3, 3)
    packed = O.pack(want["codes"]).reshape(-1)
    np.testing.assert_array_equal(c.copyTo(), packed)
    np.testing.assert_array_equal(q.mxScales, want["scales"])
    if fmt == A.NVFP4:
        assert q.mxTensorScale.tolist() == [want["t"], want["top"]]
    else:
        assert q.mxTensorScale is None

    s = q.swizzleConstant(5, 3).fold()
    total = (packed.size + 511) // 512 * 512
    np.testing.assert_array_equal(s.copyTo(), oracle.swizzle(np.pad(packed, (0, total - packed.size)), 5))

    for elem, dt in ((A.F32, np.float32), (A.F16, np.float16)):
        back = q.dequantizeMx(fmt, elem).fold()
        assert back.getType().dtype == elem and tuple(back.getType().order) == tuple(DimsOrder.OYXI)
        np.testing.assert_array_equal(back.getValues(), want["values"].astype(np.float32).astype(dt).reshape(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_swizzled_first_and_quantised_then(gpu, fmt):
    a = ContentAttr.get(np.random.default_rng(8).normal(0, 1, (24, 96)).astype(np.float16), backend=gpu)
    one, other = a.quantizeMx(fmt).swizzleConstant(5, 3), a.swizzleConstant(5, 3).quantizeMx(fmt)
    np.testing.assert_array_equal(one.fold().copyTo(), other.fold().copyTo())
    np.testing.assert_array_equal(one.mxScales, other.mxScales)
    assert (one.mxScales != 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_stored_codes_and_scales_are_read_back(gpu, fmt):
    """As a later compilation finds them: packed bytes and scales; also re-typed by the constant-folding pass, and with
    the result left on the device."""
    w = np.random.default_rng(4).normal(0, 1, (10, 96)).astype(np.float16)
    q = ContentAttr.get(w, backend=gpu).quantizeMx(fmt)
    c = q.fold()
    want = O.quantize(w.astype(np.float64), fmt)["values"].astype(np.float16)
    stored = ContentAttr.get(np.array(c.copyTo()), NDType((10, 96), A.F4E2M1), is_splat=False, backend=gpu)
    back = stored.dequantizeMx(fmt, A.F16, q.mxScales, q.mxTensorScale)
    np.testing.assert_array_equal(back.fold().getValues().reshape(10, 96), want)

    # the pass re-types packed elements as a four-dimensional constant
    q4 = ContentAttr.get(w.reshape(1, 1, 10, 96), backend=gpu).quantizeMx(fmt)
    op, = constant_folding_pass([DeclareOp(NDType((1, 1, 10, 96), A.F4E2M1), q4)])
    again = op.getContentAttr().dequantizeMx(fmt, A.F16, q.mxScales, q.mxTensorScale)
    np.testing.assert_array_equal(again.fold().getValues().reshape(10, 96), want)

    q.mxScales[:] = 0
    r = gpu.fold_resident(q._baseType, q._base, False, q.getTransformations())
    np.testing.assert_array_equal(r.to_content().copyTo(), c.copyTo())
    assert (q.mxScales != 0).any()  # written from the device
    r.release()
    r = gpu.fold_resident(stored._baseType, stored._base, False, back.getTransformations())
    np.testing.assert_array_equal(r.to_content().getValues().reshape(10, 96), want)
    r.release()


@pytest.mark.gpu
def test_given_tensor_scale_and_lazy_types(gpu):
    """A value op in front (the content is 32 bits wide, its type 16), a splat, a given tensor scale."""
    w = np.random.default_rng(5).normal(0, 1, (6, 64)).astype(np.float16)
    q = ContentAttr.get(w, backend=gpu).rescale(0.3).quantizeMx(A.NVFP4, tensorScale=0.125)
    x = (w.astype(np.float32) * np.float32(0.3)).astype(np.float16)
    want = O.quantize(x.astype(np.float64), A.NVFP4, t=0.125)
    np.testing.assert_array_equal(q.fold().copyTo(), O.pack(want["codes"]).reshape(-1))
    np.testing.assert_array_equal(q.mxScales, want["scales"])
    assert q.mxTensorScale[0] == 0.125
    s = ContentAttr.get(np.array([1.5], np.float32), NDType((4, 32), A.F32), is_splat=True, backend=gpu).quantizeMx(A.MXFP4)
    want = O.quantize(np.full((4, 32), 1.5), A.MXFP4)
    np.testing.assert_array_equal(s.fold().copyTo(), O.pack(want["codes"]).reshape(-1))


@pytest.mark.gpu
def test_what_may_not_follow(gpu):
    w = np.ones((4, 64), np.float16)
    q = ContentAttr.get(w, backend=gpu).quantizeMx(A.MXFP4)
    for a in (q.reorder((1, 0)), q.padWithZero((0, 0), (0, 32)), q.add(1.0)):
        with pytest.raises((ConstError, Unsupported)):
            a.fold()
    with pytest.raises(ValueError, match="none of a QuantizeMx"):
        q.dequantizeMx(A.NVFP4, A.F16).fold()
    b = ContentAttr.get(np.zeros(128, np.uint8), NDType((1, 1, 1, 128), A.UI8), is_splat=False, backend=gpu)
    typed = b.changeShapeAndElemType((1, 1, 4, 64), A.F4E2M1)
    with pytest.raises((ConstError, Unsupported)):
        typed.padWithZero((0,) * 4, (0, 0, 0, 32)).fold()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_batched_fold(gpu, fmt):
    """Many weights in one call, their scales kept on the device, next to an int8 constant."""
    rng = np.random.default_rng(6)
    shapes = [(64, 256), (1, 32), (33, 96), (128, 4096), (40, 11008)] * 8
    data = [rng.normal(0, 0.02, s).astype(np.float16) for s in shapes]
    decls = [ConstantDecl(f"w{i}", NDType(s, A.F16), [Q(fmt)], 2 * s[0] * s[1], compress=False) for i, s in enumerate(shapes)]
    i8 = rng.integers(-9, 9, (64, 64, 1, 1)).astype(np.int8)
    decls.append(ConstantDecl("i8", NDType(i8.shape, A.SI8), [Transform(A.X_REORDER, a=DimsOrder.NHWC)], i8.size, compress=False))
    folder = ShardFolder(gpu, decls)
    ins, sides, held = [], [], []
    for d in data + [i8]:
        ins.append(gpu.dev_alloc(d.nbytes))
        gpu.upload(ins[-1], d)
    for s in shapes:
        sides.append((gpu.dev_alloc(s[0] * -(-s[1] // O.BLOCK[fmt])), gpu.dev_alloc(8)))
    out = gpu.dev_alloc(folder.folded_bytes)
    try:
        for _ in range(2):
            gpu.fill_zero(out, folder.folded_bytes)
            folder.fold(ins, out, side_ptrs=sides + [None])
            gpu.synchronize()
            blob = gpu.download(out, folder.folded_bytes)
        for i, s in enumerate(shapes[:5] + shapes[-1:]):
            i = i if i < 5 else len(shapes) - 1
            want = O.quantize(data[i].astype(np.float64), fmt)
            got = blob[folder.folded_offsets[i]:][:folder.folded_sizes[i]]
            np.testing.assert_array_equal(got, O.pack(want["codes"]).reshape(-1))
            np.testing.assert_array_equal(gpu.download(sides[i][0], want["scales"].size), want["scales"].reshape(-1))
            if fmt == A.NVFP4:
                assert gpu.download(sides[i][1], 8).view(np.float32).tolist() == [want["t"], want["top"]]
        got = blob[folder.folded_offsets[-1]:][:i8.size]
        np.testing.assert_array_equal(got.view(np.int8), i8.reshape(-1))
    finally:
        for p in ins + [x for s in sides for x in s] + [out]:
            gpu.dev_free(p)


@pytest.mark.gpu
def test_weights_are_taken_if_the_layer_can_bear_it(gpu):
    rng = np.random.default_rng(7)
    w = rng.normal(0, 0.05, (48, 256)).astype(np.float16)
    x = rng.normal(0, 1, (30, 256)).astype(np.float16)
    y = x.astype(np.float64) @ w.astype(np.float64).T
    weights = ContentAttr.get(w, backend=gpu)

    def error(fmt):
        qx, qw = O.quantize(x.astype(np.float64), fmt)["values"], O.quantize(w.astype(np.float64), fmt)["values"]
        return np.linalg.norm(qx @ qw.T - y) / np.linalg.norm(y)
    nv, mxe = error(A.NVFP4), error(A.MXFP4)
    a, fmt, e = chains.mx_weights(weights, x, y, tolerance=1.0)
    assert fmt == A.NVFP4 and abs(e - nv) < 1e-5 * 300 ** 0.5  # sums of 256 products in 32 bits
    assert a.getType().dtype == A.F4E2M1
    a, fmt, e = chains.mx_weights(weights, x.astype(np.float32), y, tolerance=1.0, formats=(A.MXFP4,))
    assert fmt == A.MXFP4 and abs(e - mxe) < 2e-4
    a, fmt, e = chains.mx_weights(weights, x, y, tolerance=min(nv, mxe) / 2)
    assert a is weights and fmt is None and abs(e - min(nv, mxe)) < 2e-4
    with pytest.raises(ValueError):
        chains.mx_weights(weights, x[:, :128], y, tolerance=1.0)
    with pytest.raises(ConstError):
        chains.mx_weights(ContentAttr.get(w[:, :40], backend=gpu), x[:, :40], y, tolerance=1.0)
