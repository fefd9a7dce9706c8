// Block-scaled 4-bit quantisation and its inverse (formats and storage: include/b200const.h).
//
// Every thread has 8 neighbours of a row: one 16-byte load of 16-bit elements, one 4-byte word of codes.
// Four threads (mxfp4) or two (nvfp4) share a block and find its largest magnitude with shuffles.
#include "mx.h"
#include "runtime.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace b200c {

namespace {

struct MxQuantParams {
    const void* src;
    long long srcLd;
    long long rows, cols;
    unsigned char* codes;
    long long ld;
    unsigned char* scales;
    int tiled;
    float* tensorScale;
    int scaleGiven;
    void* values;  // or nullptr
    long long valuesLd;
    long long blocks;       // blocks of a row
    long long scaleRows;    // rows of scale bytes, those that fill up the last tile included
    long long scaleBlocks;  // the same for blocks
    int wideIn, wideValues;  // 16-byte accesses are aligned
};

struct MxDequantParams {
    const unsigned char* codes;
    long long ld;
    const unsigned char* scales;
    int tiled;
    const float* tensorScale;
    long long rows, cols, blocks;
    void* out;
    long long outLd;
    int wideOut;
};

__device__ __forceinline__ long long scaleAt(int tiled, long long row, long long block, long long blocks) {
    if (!tiled) return row * blocks + block;
    const long long chunk = (row >> 7) * ((blocks + 3) >> 2) + (block >> 2);
    return chunk * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

template <class T>
__device__ __forceinline__ float toFloat(T v);
template <>
__device__ __forceinline__ float toFloat<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float toFloat<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float toFloat<float>(float v) {
    return v;
}
template <class T>
__device__ __forceinline__ T fromFloat(float v);
template <>
__device__ __forceinline__ __half fromFloat<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float fromFloat<float>(float v) {
    return v;
}

// two 32-bit values -> two codes in a byte, `lo` in the low nibble: nearest even, at most 6
__device__ __forceinline__ unsigned int codePair(float lo, float hi) {
    unsigned int r;
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
// a byte of two codes -> their values in f16 (exact)
__device__ __forceinline__ float2 codeValues(unsigned int byte) {
    unsigned int h;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ unsigned int toE4m3(float v) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
    return r & 0xFFu;
}
__device__ __forceinline__ float fromE4m3(unsigned int byte) {
    unsigned int h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(byte)));
    return __low2float(*reinterpret_cast<__half2*>(&h));
}
// 2^X of the byte X + 127; 2^-127 is a subnormal number, 0xFF is NaN
__device__ __forceinline__ float fromE8m0(unsigned int byte) {
    return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, bool wide, long long left, float v[8]) {
    if (wide && left >= 8) {
        alignas(16) T t[8];
        constexpr int n = 8 * sizeof(T) / 16;
#pragma unroll
        for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = toFloat<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? toFloat<T>(p[i]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, bool wide, long long left, const float v[8]) {
    if (wide && left >= 8) {
        alignas(16) T t[8];
        constexpr int n = 8 * sizeof(T) / 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = fromFloat<T>(v[i]);
#pragma unroll
        for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = fromFloat<T>(v[i]);
    }
}

// the smallest power of two t >= 2^-126 with top <= 2688 t; 2688 = 1.3125 * 2^11, so t = 2^(e - 11) when top's
// significand is at most 1.3125 and twice that otherwise
__device__ __forceinline__ float tensorScaleOf(float top) {
    if (!(top > 0.f)) return 1.f;
    const unsigned int bits = __float_as_uint(top);
    int e = static_cast<int>(bits >> 23) - 11 + ((bits & 0x7FFFFFu) > 0x280000u ? 1 : 0);
    return __uint_as_float(static_cast<unsigned int>(max(e, 1)) << 23);
}

// largest finite magnitude of the matrix -> tensorScale[1] (zeroed before).  Magnitudes compare like
// their bits, and a maximum does not depend on the order it is taken in.
template <class T>
__global__ void __launch_bounds__(256) mxTopKernel(const __grid_constant__ MxQuantParams p) {
    unsigned int top = 0;
    const long long units = (p.cols + 7) / 8;
    for (long long r = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; r < p.rows; r += static_cast<long long>(gridDim.y) * blockDim.y) {
        const T* row = static_cast<const T*>(p.src) + r * p.srcLd;
        for (long long u = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; u < units; u += static_cast<long long>(gridDim.x) * blockDim.x) {
            float v[8];
            load8<T>(row + u * 8, p.wideIn != 0, p.cols - u * 8, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned int a = __float_as_uint(v[i]) & 0x7FFFFFFFu;
                if (a < 0x7F800000u) top = max(top, a);
            }
        }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (((threadIdx.y * blockDim.x + threadIdx.x) & 31) == 0 && top) atomicMax(reinterpret_cast<unsigned int*>(p.tensorScale) + 1, top);
}

template <class T, bool NV>
__global__ void __launch_bounds__(256) mxQuantKernel(const __grid_constant__ MxQuantParams p) {
    float t = 1.f;
    if (NV) {
        if (p.scaleGiven) {
            t = p.tensorScale[0];
        } else {
            t = tensorScaleOf(p.tensorScale[1]);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && threadIdx.y == 0) p.tensorScale[0] = t;
        }
    }
    constexpr int lanes = NV ? 2 : 4;  // threads of a block
    const long long units = (p.cols + 31) / 32 * 4;               // words of codes in a row
    const long long all = max(units, p.scaleBlocks * lanes);      // and those that only write a tile's filling scales
    for (long long r = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; r < p.scaleRows; r += static_cast<long long>(gridDim.y) * blockDim.y) {
        const T* row = static_cast<const T*>(p.src) + r * p.srcLd;
        // a group of four threads runs the loop together: `all` and blockDim.x are multiples of 4
        for (long long u = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; u < all; u += static_cast<long long>(gridDim.x) * blockDim.x) {
            float v[8];
            const long long left = r < p.rows ? p.cols - u * 8 : 0;
            load8<T>(row + u * 8, p.wideIn != 0, left, v);
            unsigned int top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            const unsigned int group = 0xFu << (((threadIdx.y * blockDim.x + threadIdx.x) & 31) & ~3);
            top = max(top, __shfl_xor_sync(group, top, 1));
            if (!NV) top = max(top, __shfl_xor_sync(group, top, 2));

            const bool poison = top >= 0x7F800000u;  // a NaN or an infinity in the block
            unsigned int scale;
            float d, q[8];
            bool zero = poison;
            if (!NV) {
                // the exponent field of the largest magnitude, less 2; subnormal numbers have the field 0
                scale = poison ? 0xFFu : static_cast<unsigned int>(max(static_cast<int>(top >> 23) - 2, 0));
                d = fromE8m0(scale);
                const float up = __uint_as_float((254u - min(scale, 253u)) << 23);  // 2^-X
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = v[i] * up;
            } else {
                // 0 / 0 and a NaN t fall to the scale NaN
                const float s = __fdiv_rn(__uint_as_float(top), 6.f * t);
                scale = poison || !(t > 0.f) || !(t <= 3.402823466e38f) ? 0x7Fu : toE4m3(fminf(s, 448.f));
                d = __fmul_rn(fromE4m3(scale), t);
                zero = scale == 0x7Fu || !(d > 0.f);
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[i], d);
            }
            unsigned int word = 0;
            if (!zero) {
#pragma unroll
                for (int i = 0; i < 4; ++i) word |= codePair(q[2 * i], q[2 * i + 1]) << (8 * i);
            }
            if (r < p.rows && u < units) *reinterpret_cast<unsigned int*>(p.codes + r * p.ld + u * 4) = word;
            if ((u & (lanes - 1)) == 0) {
                const long long b = u / lanes;
                if (b < p.scaleBlocks) p.scales[scaleAt(p.tiled, r, b, p.blocks)] = static_cast<unsigned char>(left > 0 ? scale : 0u);
            }
            if (p.values && left > 0) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 c = codeValues((word >> (8 * i)) & 0xFFu);
                    w[2 * i] = c.x * d;
                    w[2 * i + 1] = c.y * d;
                }
                store8<T>(static_cast<T*>(p.values) + r * p.valuesLd + u * 8, p.wideValues != 0, left, w);
            }
        }
    }
}

template <class T, bool NV>
__global__ void __launch_bounds__(256) mxDequantKernel(const __grid_constant__ MxDequantParams p) {
    const float t = NV ? p.tensorScale[0] : 1.f;
    const long long units = (p.cols + 7) / 8;
    for (long long r = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; r < p.rows; r += static_cast<long long>(gridDim.y) * blockDim.y) {
        for (long long u = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; u < units; u += static_cast<long long>(gridDim.x) * blockDim.x) {
            const unsigned int word = *reinterpret_cast<const unsigned int*>(p.codes + r * p.ld + u * 4);
            const unsigned int scale = p.scales[scaleAt(p.tiled, r, u / (NV ? 2 : 4), p.blocks)];
            const float d = NV ? __fmul_rn(fromE4m3(scale), t) : fromE8m0(scale);
            float w[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 c = codeValues((word >> (8 * i)) & 0xFFu);
                w[2 * i] = c.x * d;
                w[2 * i + 1] = c.y * d;
            }
            store8<T>(static_cast<T*>(p.out) + r * p.outLd + u * 8, p.wideOut != 0, p.cols - u * 8, w);
        }
    }
}

// rows x units of 8 elements over CTAs of 256 threads; threads of a CTA cover as much of a row as there is
void gridFor(Context* ctx, long long rows, long long units, dim3* grid, dim3* block) {
    unsigned int x = 4;
    while (x < 256 && x < units) x *= 2;
    *block = dim3(x, 256 / x);
    const long long gx = std::max<long long>(1, std::min<long long>((units + x - 1) / x, 1024));
    const long long want = (rows + block->y - 1) / block->y;
    const long long most = std::max<long long>(1, ctx->smCount * 64LL / gx);
    *grid = dim3(static_cast<unsigned int>(gx), static_cast<unsigned int>(std::max<long long>(1, std::min<long long>(want, std::min<long long>(most, 65535)))));
}

bool aligned16(const void* p, long long ldBytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ldBytes % 16 == 0;
}

template <class T>
void quantizeAs(Context* ctx, const MxQuantParams& p, bool nv) {
    dim3 grid, block;
    if (nv && !p.scaleGiven) {
        fillBytes(ctx, p.tensorScale, 0, 8);
        if (p.rows > 0 && p.cols > 0) {
            gridFor(ctx, p.rows, (p.cols + 7) / 8, &grid, &block);
            mxTopKernel<T><<<grid, block, 0, ctx->stream>>>(p);
            B2_CUDA(cudaGetLastError());
            ++ctx->launches;
        }
    }
    // an empty matrix has no scales, but its factor is still written
    const long long units = std::max((p.cols + 31) / 32 * 4, p.scaleBlocks * (nv ? 2 : 4));
    if ((p.scaleRows == 0 || units == 0) && !(nv && !p.scaleGiven)) return;
    gridFor(ctx, p.scaleRows, units, &grid, &block);
    if (nv) {
        mxQuantKernel<T, true><<<grid, block, 0, ctx->stream>>>(p);
    } else {
        mxQuantKernel<T, false><<<grid, block, 0, ctx->stream>>>(p);
    }
    B2_CUDA(cudaGetLastError());
    ++ctx->launches;
}

template <class T>
void dequantizeAs(Context* ctx, const MxDequantParams& p, bool nv) {
    dim3 grid, block;
    gridFor(ctx, p.rows, (p.cols + 7) / 8, &grid, &block);
    if (nv) {
        mxDequantKernel<T, true><<<grid, block, 0, ctx->stream>>>(p);
    } else {
        mxDequantKernel<T, false><<<grid, block, 0, ctx->stream>>>(p);
    }
    B2_CUDA(cudaGetLastError());
    ++ctx->launches;
}

}  // namespace

void launchMxQuantize(Context* ctx, const void* src, int dtype, int64_t srcLd, const b200c_mx_matrix& out, void* values,
                      int64_t valuesLd, bool scaleGiven) {
    const int es = dtBits(dtype) / 8;
    MxQuantParams p;
    p.src = src;
    p.srcLd = srcLd;
    p.rows = out.rows;
    p.cols = out.cols;
    p.codes = static_cast<unsigned char*>(out.codes);
    p.ld = out.ld;
    p.scales = static_cast<unsigned char*>(out.scales);
    p.tiled = out.scale_layout == B200C_MX_SCALES_TILED;
    p.tensorScale = out.tensor_scale;
    p.scaleGiven = scaleGiven;
    p.values = values;
    p.valuesLd = valuesLd;
    p.blocks = mxBlocks(out.format, out.cols);
    p.scaleRows = out.cols == 0 ? 0 : p.tiled ? roundUp(out.rows, 128) : out.rows;
    p.scaleBlocks = p.tiled ? roundUp(p.blocks, 4) : p.blocks;
    p.wideIn = aligned16(src, srcLd * es);
    p.wideValues = values && aligned16(values, valuesLd * es);
    const bool nv = out.format == B200C_NVFP4;
    if (dtype == B200C_F16) {
        quantizeAs<__half>(ctx, p, nv);
    } else if (dtype == B200C_BF16) {
        quantizeAs<__nv_bfloat16>(ctx, p, nv);
    } else {
        quantizeAs<float>(ctx, p, nv);
    }
}

void launchMxDequantize(Context* ctx, const b200c_mx_matrix& m, void* out, int dtype, int64_t outLd) {
    if (m.rows == 0 || m.cols == 0) return;
    MxDequantParams p;
    p.codes = static_cast<const unsigned char*>(m.codes);
    p.ld = m.ld;
    p.scales = static_cast<const unsigned char*>(m.scales);
    p.tiled = m.scale_layout == B200C_MX_SCALES_TILED;
    p.tensorScale = m.tensor_scale;
    p.rows = m.rows;
    p.cols = m.cols;
    p.blocks = mxBlocks(m.format, m.cols);
    p.out = out;
    p.outLd = outLd;
    p.wideOut = aligned16(out, outLd * (dtBits(dtype) / 8));
    const bool nv = m.format == B200C_NVFP4;
    if (dtype == B200C_F16) {
        dequantizeAs<__half>(ctx, p, nv);
    } else if (dtype == B200C_BF16) {
        dequantizeAs<__nv_bfloat16>(ctx, p, nv);
    } else {
        dequantizeAs<float>(ctx, p, nv);
    }
}

}  // namespace b200c
