// Sizes of block-scaled 4-bit matrices and the checks of the calls that take them: host code.
#include "mx.h"

#include <string>

namespace b200c {

namespace {

// A row or column index fits 31 bits with room to round up to a tile; offsets are 64 bits everywhere.
constexpr int64_t kMaxExtent = 0x7FFFFFFF - 65536;

struct Range {
    const char* what;
    uintptr_t lo, hi;
};

Range rangeOf(const char* what, const void* p, int64_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return Range{what, a, a + static_cast<uintptr_t>(bytes > 0 ? bytes : 0)};
}

void checkApart(const Range& out, const Range& other) {
    if (out.lo < out.hi && other.lo < other.hi && out.lo < other.hi && other.lo < out.hi) {
        throw BadArg(std::string(out.what) + " overlaps " + other.what);
    }
}

int64_t spanBytes(int64_t rows, int64_t ld, int64_t cols, int64_t elem) {
    return rows > 0 && cols > 0 ? ((rows - 1) * ld + cols) * elem : 0;
}

int elemBytes(int dtype) {
    switch (dtype) {
    case B200C_F16:
    case B200C_BF16:
        return 2;
    case B200C_F32:
        return 4;
    default:
        throw BadArg("the element type has to be f16, bf16 or f32");
    }
}

// a dense side of a call: rows x cols of `dtype`, ld elements between rows
Range checkDense(const char* what, const void* p, int dtype, int64_t rows, int64_t cols, int64_t ld) {
    const int es = elemBytes(dtype);
    if (ld < cols) throw BadArg(std::string(what) + ": fewer elements between rows than columns");
    if (rows > 0 && ld > (INT64_MAX / 8) / rows) throw BadArg(std::string(what) + ": the distance between rows is too large");
    if (rows > 0 && cols > 0) {
        if (!p) throw BadArg(std::string(what) + ": null pointer");
        if (reinterpret_cast<uintptr_t>(p) % es) throw BadArg(std::string(what) + ": not aligned to its element type");
    }
    return rangeOf(what, p, spanBytes(rows, ld, cols, es));
}

struct MatrixRanges {
    Range codes, scales, tensor;
};

MatrixRanges checkMatrix(const char* what, const b200c_mx_matrix* m) {
    if (!m) throw BadArg(std::string(what) + ": null descriptor");
    mxCheckShape(m->format, m->scale_layout, m->rows, m->cols);
    const std::string name(what);
    if (m->ld % 16 != 0 || m->ld < mxPitch(m->cols)) {
        throw BadArg(name + ": the bytes between rows of codes have to be a multiple of 16 and hold the columns rounded up to 32");
    }
    if (m->rows > 0 && m->ld > (INT64_MAX / 8) / m->rows) throw BadArg(name + ": the distance between rows is too large");
    const bool any = m->rows > 0 && m->cols > 0;
    if (any && (!m->codes || !m->scales)) throw BadArg(name + ": null pointer");
    if (any && reinterpret_cast<uintptr_t>(m->codes) % 16) throw BadArg(name + ": codes have to be 16-byte aligned");
    if (any && m->scale_layout == B200C_MX_SCALES_TILED && reinterpret_cast<uintptr_t>(m->scales) % 16) {
        throw BadArg(name + ": tiled scales have to be 16-byte aligned");
    }
    const bool tensor = m->format == B200C_NVFP4;
    if (tensor && !m->tensor_scale) throw BadArg(name + ": nvfp4 needs a tensor scale");
    if (tensor && reinterpret_cast<uintptr_t>(m->tensor_scale) % 4) throw BadArg(name + ": the tensor scale is not aligned");
    return MatrixRanges{rangeOf("codes", m->codes, spanBytes(m->rows, m->ld, mxPitch(m->cols), 1)),
                        rangeOf("scales", m->scales, mxScaleBytes(m->format, m->scale_layout, m->rows, m->cols)),
                        rangeOf("tensor scale", m->tensor_scale, tensor ? 8 : 0)};
}

}  // namespace

int64_t mxScaleBytes(int format, int layout, int64_t rows, int64_t cols) {
    const int64_t blocks = mxBlocks(format, cols);
    if (layout == B200C_MX_SCALES_ROWS) return rows * blocks;
    return (rows + 127) / 128 * ((blocks + 3) / 4) * 512;
}

void mxCheckShape(int format, int layout, int64_t rows, int64_t cols) {
    if (format != B200C_MXFP4 && format != B200C_NVFP4) throw BadArg("unknown block-scaled format");
    if (layout != B200C_MX_SCALES_ROWS && layout != B200C_MX_SCALES_TILED) throw BadArg("unknown layout of scales");
    if (rows < 0 || cols < 0) throw BadArg("negative dimension");
    if (rows > kMaxExtent || cols > kMaxExtent) throw BadArg("dimension too large");
}

void mxCheckQuantize(const void* src, int dtype, int64_t srcLd, const b200c_mx_matrix* out, const void* values,
                     int64_t valuesLd, int flags) {
    if (flags & ~B200C_MX_SCALE_GIVEN) throw BadArg("unknown flags");
    const MatrixRanges m = checkMatrix("quantised matrix", out);
    if ((flags & B200C_MX_SCALE_GIVEN) && out->format != B200C_NVFP4) throw BadArg("mxfp4 has no tensor scale to give");
    const Range in = checkDense("source", src, dtype, out->rows, out->cols, srcLd);
    const Range val = values ? checkDense("values", values, dtype, out->rows, out->cols, valuesLd) : Range{"values", 0, 0};
    checkApart(m.codes, in);
    checkApart(m.scales, in);
    checkApart(m.tensor, in);
    checkApart(val, in);
    checkApart(m.codes, m.scales);
    checkApart(m.codes, m.tensor);
    checkApart(m.scales, m.tensor);
    checkApart(val, m.codes);
    checkApart(val, m.scales);
    checkApart(val, m.tensor);
}

void mxCheckDequantize(const b200c_mx_matrix* m, const void* out, int dtype, int64_t outLd) {
    const MatrixRanges in = checkMatrix("quantised matrix", m);
    const Range dst = checkDense("output", out, dtype, m->rows, m->cols, outLd);
    checkApart(dst, in.codes);
    checkApart(dst, in.scales);
    checkApart(dst, in.tensor);
}

void mxCheckMatmul(const b200c_mx_matrix* a, const b200c_mx_matrix* b, const void* out, int dtype, int64_t outLd) {
    const MatrixRanges ra = checkMatrix("left matrix", a), rb = checkMatrix("right matrix", b);
    if (a->format != b->format) throw BadArg("the two matrices have different formats");
    if (a->cols != b->cols) throw BadArg("the two matrices have different numbers of columns");
    if (a->scale_layout != B200C_MX_SCALES_TILED || b->scale_layout != B200C_MX_SCALES_TILED) {
        throw BadArg("the product reads tiled scales");
    }
    // the loads' descriptors hold distances below 2^40 bytes
    if (a->ld >= (int64_t(1) << 40) || b->ld >= (int64_t(1) << 40)) throw BadArg("the distance between rows of codes is too large for a product");
    const Range dst = checkDense("output", out, dtype, a->rows, b->rows, outLd);
    for (const MatrixRanges* m : {&ra, &rb}) {
        checkApart(dst, m->codes);
        checkApart(dst, m->scales);
        checkApart(dst, m->tensor);
    }
}

}  // namespace b200c
