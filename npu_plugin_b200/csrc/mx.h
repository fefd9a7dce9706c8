// Block-scaled 4-bit matrices: descriptors, sizes and the checks of their arguments (mx.cpp), and the
// launchers of the kernels (mx_kernels.cu, mx_matmul.cu).  Formats and storage: include/b200const.h.
#pragma once

#include "../../include/b200const.h"
#include "ctype.h"

#include <cstddef>
#include <cstdint>

namespace b200c {

struct Context;

inline int mxBlock(int format) {
    return format == B200C_MXFP4 ? 32 : 16;
}
inline int64_t mxBlocks(int format, int64_t cols) {
    return (cols + mxBlock(format) - 1) / mxBlock(format);
}
// bytes of a row of codes: whole groups of 32 elements
inline int64_t mxPitch(int64_t cols) {
    return (cols + 31) / 32 * 16;
}
int64_t mxScaleBytes(int format, int layout, int64_t rows, int64_t cols);

// Throw BadArg for what the header does not allow; no device is touched.
void mxCheckShape(int format, int layout, int64_t rows, int64_t cols);
void mxCheckQuantize(const void* src, int dtype, int64_t srcLd, const b200c_mx_matrix* out, const void* values,
                     int64_t valuesLd, int flags);
void mxCheckDequantize(const b200c_mx_matrix* m, const void* out, int dtype, int64_t outLd);
void mxCheckMatmul(const b200c_mx_matrix* a, const b200c_mx_matrix* b, const void* out, int dtype, int64_t outLd);

void launchMxQuantize(Context* ctx, const void* src, int dtype, int64_t srcLd, const b200c_mx_matrix& out, void* values,
                      int64_t valuesLd, bool scaleGiven);
void launchMxDequantize(Context* ctx, const b200c_mx_matrix& m, void* out, int dtype, int64_t outLd);
void launchMxMatmul(Context* ctx, const b200c_mx_matrix& a, const b200c_mx_matrix& b, void* out, int dtype, int64_t outLd);

}  // namespace b200c
