// Product of two block-scaled 4-bit matrices, out = A B^T, on the tensor cores (formats and storage:
// include/b200const.h).
//
// sum_k A[i][k] B[j][k] with A[i][k] = code * scale: tcgen05.mma takes the codes from shared memory and the
// scales from tensor memory and multiplies both in, 64 elements of k at a time; sums are 32 bits wide.
// One side's rows are the 128 rows of a tile ("P"), the other's its columns ("Q"); the wider side is P when
// the other has few rows, since 128 is the only height there is.
#include "mx.h"
#include "runtime.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

namespace b200c {

namespace {

struct MxMatmulParams {
    const unsigned char* scalesP;
    const unsigned char* scalesQ;
    const float* tensorP;  // nullptr: 1
    const float* tensorQ;
    long long rowsP, rowsQ, k;
    long long chunks;      // tiles of 4 blocks along k: 512 bytes of scales each, per 128 rows
    int scaleTilesQ;       // tiles of 128 rows that the Q side's scales have
    int ktiles;
    int tilesQ;
    void* out;
    long long ld;
    int outTag;            // T_F16, T_BF16, T_F32
    int across;            // out[q * ld + p] instead of out[p * ld + q]
    int wide;              // 16-byte stores along a row are aligned
    int* err;
};

constexpr int kTileK = 256;      // elements of k per stage: 128 bytes of codes, one swizzle row
constexpr int kStepK = 64;       // elements of k per tcgen05.mma
constexpr int kThreads = 192;    // warps 0-3: epilogue, 4: loads, 5: mma

template <int BN, bool NV>
struct Tile {
    static constexpr int chunksPerTile = NV ? 4 : 2;  // 512-byte tiles of scales per stage and 128 rows
    static constexpr int rowTilesQ = (BN + 127) / 128;
    static constexpr int bytesP = 128 * 128;
    static constexpr int bytesQ = BN * 128;
    static constexpr int scaleBytesP = chunksPerTile * 512;
    static constexpr int scaleBytesQ = scaleBytesP * rowTilesQ;
    static constexpr int stageBytes = (bytesP + bytesQ + scaleBytesP + scaleBytesQ + 1023) / 1024 * 1024;
    static constexpr int stages = 4;
    static constexpr int smemBytes = 1024 /* barriers */ + 1024 /* alignment */ + stages * stageBytes;
    static constexpr int scaleCols = chunksPerTile * 4 * (1 + rowTilesQ);  // tensor memory columns of a stage's scales
    static constexpr int needCols = BN + 2 * scaleCols;
    static constexpr int cols = needCols <= 32 ? 32 : needCols <= 64 ? 64 : needCols <= 128 ? 128 : needCols <= 256 ? 256 : 512;
};

__device__ __forceinline__ unsigned int smemAddr(const void* p) {
    return static_cast<unsigned int>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void barInit(unsigned int bar, unsigned int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ bool barTry(unsigned int bar, unsigned int parity) {
    unsigned int done;
    asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
    return done != 0;
}
// Every wait ends: after two seconds it gives up, and so do the others once one has.
__device__ __noinline__ bool barWaitSlow(unsigned int bar, unsigned int parity, volatile int* stalled) {
    const long long start = clock64();
    while (!barTry(bar, parity)) {
        if (*stalled || clock64() - start > 4000000000ll) {
            *stalled = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool barWait(unsigned int bar, unsigned int parity, volatile int* stalled) {
    if (barTry(bar, parity)) return true;
    return barWaitSlow(bar, parity, stalled);
}

__device__ __forceinline__ void loadTile(unsigned int dst, const CUtensorMap* map, int x, int y, unsigned int bar) {
    asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void loadBytes(unsigned int dst, const void* src, unsigned int bytes, unsigned int bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// Shared memory descriptor of a K-major operand in rows of 128 bytes, swizzled over 128 bytes: groups of 8 rows
// are 1024 bytes apart.
__device__ __forceinline__ unsigned long long operandDesc(unsigned int addr) {
    return static_cast<unsigned long long>((addr & 0x3FFFF) >> 4) | (1ull << 16) | (static_cast<unsigned long long>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// The same for a 512-byte tile of scales, 32 rows of 16 bytes without a swizzle: groups of 8 rows 128 bytes apart.
__device__ __forceinline__ unsigned long long scaleDesc(unsigned int addr) {
    return static_cast<unsigned long long>((addr & 0x3FFFF) >> 4) | (static_cast<unsigned long long>(128 >> 4) << 32) | (1ull << 46);
}
// 32 rows x 16 bytes -> 4 columns of tensor memory, the same in each quarter of the lanes
__device__ __forceinline__ void copyScales(unsigned int tmem, unsigned long long desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

template <bool NV>
__device__ __forceinline__ void mma(unsigned int d, unsigned long long a, unsigned long long b, unsigned int idesc,
                                    unsigned int scaleA, unsigned int scaleB, unsigned int accumulate) {
    if (NV) {
        asm volatile(
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
                "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate)
                : "memory");
    } else {
        asm volatile(
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
                "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate)
                : "memory");
    }
}
// arrives at `bar` once everything issued so far by this thread to the tensor core is done
__device__ __forceinline__ void mmaCommit(unsigned int bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Instruction descriptor: e2m1 x e2m1, 128 x BN; the scales' type in bit 23 (1: e8m0); which pair of a word's
// four scale bytes is meant in bits 29 (A) and 4 (B).
template <int BN, bool NV>
__device__ __forceinline__ unsigned int instruction(int pair) {
    return (1u << 7) | (1u << 10) | (static_cast<unsigned int>(BN >> 3) << 17) | (NV ? 0u : 1u << 23) | (1u << 27) |
           (static_cast<unsigned int>(pair) << 29) | (static_cast<unsigned int>(pair) << 4);
}

__device__ __forceinline__ void readColumns(unsigned int addr, float v[32]) {
    unsigned int r[32];
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
              "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
              "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(addr)
            : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void readColumns16(unsigned int addr, float v[32]) {
    unsigned int r[16];
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(addr)
            : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

template <class T>
__device__ __forceinline__ T toOut(float v);
template <>
__device__ __forceinline__ __half toOut<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 toOut<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float toOut<float>(float v) {
    return v;
}

// N accumulator columns of row p, columns q0.. of the product
template <class T, int N>
__device__ __forceinline__ void storeColumns(const MxMatmulParams& g, long long p, long long q0, const float* v) {
    if (p >= g.rowsP) return;
    const long long left = g.rowsQ - q0;
    T* out = static_cast<T*>(g.out);
    if (g.across) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) out[(q0 + i) * g.ld + p] = toOut<T>(v[i]);
        return;
    }
    T* row = out + p * g.ld + q0;
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N; i += per) {
        if (g.wide && i + per <= left) {
            alignas(16) T t[per];
#pragma unroll
            for (int j = 0; j < per; ++j) t[j] = toOut<T>(v[i + j]);
            *reinterpret_cast<uint4*>(row + i) = *reinterpret_cast<const uint4*>(t);
        } else {
#pragma unroll
            for (int j = 0; j < per; ++j)
                if (i + j < left) row[i + j] = toOut<T>(v[i + j]);
        }
    }
}

template <class T, int BN>
__device__ __forceinline__ void epilogue(const MxMatmulParams& g, unsigned int acc, long long p, long long q0, float alpha) {
    constexpr int n = BN < 32 ? BN : 32;
#pragma unroll 1
    for (int c = 0; c < BN; c += n) {
        float v[32];
        if (n == 32) {
            readColumns(acc + c, v);
        } else {
            readColumns16(acc + c, v);
        }
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = v[i] * alpha;
        storeColumns<T, n>(g, p, q0 + c, v);
    }
}

template <int BN, bool NV>
__global__ void __launch_bounds__(kThreads) mxMatmulKernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
                                                           const __grid_constant__ MxMatmulParams g) {
    typedef Tile<BN, NV> S;
    extern __shared__ unsigned char raw[];
    __shared__ unsigned long long bars[2 * S::stages + 1];
    __shared__ unsigned int tmemBase;
    __shared__ int stalledWord;
    volatile int* stalled = &stalledWord;
    const unsigned int stage0 = (smemAddr(raw) + 1023u) & ~1023u;
    const unsigned int full = smemAddr(bars), empty = full + 8 * S::stages, done = empty + 8 * S::stages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long p0 = static_cast<long long>(blockIdx.x / g.tilesQ) * 128;
    const long long q0 = static_cast<long long>(blockIdx.x % g.tilesQ) * BN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::stages; ++s) {
            barInit(full + 8 * s, 1);
            barInit(empty + 8 * s, 1);
        }
        barInit(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        stalledWord = 0;
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemBase)), "r"(S::cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned int acc = tmemBase, scaleCol = tmemBase + BN;

    if (warp == 4 && lane == 0) {
        const int scaleTileP = static_cast<int>(p0 / 128), scaleTileQ = static_cast<int>(q0 / 128);
        const int tilesQ = min(S::rowTilesQ, g.scaleTilesQ - scaleTileQ);  // rows behind the last tile have no scales
        int issued = 0;
        for (int kt = 0; kt < g.ktiles; ++kt) {
            const int s = kt % S::stages;
            if (kt >= S::stages && !barWait(empty + 8 * s, ((kt / S::stages) & 1) ^ 1, stalled)) break;
            const unsigned int at = stage0 + s * S::stageBytes, bar = full + 8 * s;
            const long long chunk = static_cast<long long>(kt) * S::chunksPerTile;
            const unsigned int scaleBytes = static_cast<unsigned int>(min(static_cast<long long>(S::chunksPerTile), g.chunks - chunk)) * 512u;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                         "r"(S::bytesP + S::bytesQ + scaleBytes * (1 + tilesQ))
                         : "memory");
            loadTile(at, &mapP, kt * 128, static_cast<int>(p0), bar);
            loadTile(at + S::bytesP, &mapQ, kt * 128, static_cast<int>(q0), bar);
            const unsigned int sp = at + S::bytesP + S::bytesQ;
            loadBytes(sp, g.scalesP + (scaleTileP * g.chunks + chunk) * 512, scaleBytes, bar);
            for (int i = 0; i < tilesQ; ++i) {
                loadBytes(sp + S::scaleBytesP * (1 + i), g.scalesQ + ((scaleTileQ + i) * g.chunks + chunk) * 512, scaleBytes, bar);
            }
            issued = kt + 1;
        }
        // a wait that gave up leaves copies in flight: they write this CTA's memory, so it stays until they have
        if (*stalled) {
            for (int kt = max(0, issued - S::stages); kt < issued; ++kt) {
                const long long start = clock64();
                while (!barTry(full + 8 * (kt % S::stages), (kt / S::stages) & 1) && clock64() - start < 4000000000ll) {
                }
            }
        }
    } else if (warp == 5 && lane == 0) {
        bool ok = true;
        for (int kt = 0; kt < g.ktiles; ++kt) {
            const int s = kt % S::stages;
            ok = barWait(full + 8 * s, (kt / S::stages) & 1, stalled);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned int at = stage0 + s * S::stageBytes;
            const unsigned int sp = at + S::bytesP + S::bytesQ;
            const unsigned int colP = scaleCol + (kt & 1) * S::scaleCols, colQ = colP + S::chunksPerTile * 4;
            const long long leftK = g.k - static_cast<long long>(kt) * kTileK;
            const int steps = static_cast<int>(min(static_cast<long long>(kTileK / kStepK), (leftK + kStepK - 1) / kStepK));
            const int chunks = static_cast<int>(min(static_cast<long long>(S::chunksPerTile), g.chunks - static_cast<long long>(kt) * S::chunksPerTile));
            for (int c = 0; c < chunks; ++c) {
                copyScales(colP + c * 4, scaleDesc(sp + c * 512));
                for (int i = 0; i < S::rowTilesQ; ++i) {
                    copyScales(colQ + (c * S::rowTilesQ + i) * 4, scaleDesc(sp + S::scaleBytesP * (1 + i) + c * 512));
                }
            }
            const unsigned long long dp = operandDesc(at), dq = operandDesc(at + S::bytesP);
            for (int i = 0; i < steps; ++i) {
                // mxfp4: a word of four scales reaches over 128 elements, two steps; nvfp4: over one
                const int c = NV ? i : i >> 1, pair = NV ? 0 : (i & 1) * 2;
                mma<NV>(acc, dp + i * 2, dq + i * 2, instruction<BN, NV>(pair), colP + c * 4, colQ + c * 4 * S::rowTilesQ,
                        kt > 0 || i > 0);
            }
            mmaCommit(empty + 8 * s);
        }
        mmaCommit(done);
    } else if (warp < 4) {
        const bool finished = barWait(done, 0, stalled) && !*stalled;
        if (__all_sync(0xFFFFFFFFu, finished)) {  // the reads below are the whole warp's
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float alpha = g.tensorP ? g.tensorP[0] * g.tensorQ[0] : 1.f;
            const unsigned int mine = acc + (static_cast<unsigned int>(warp * 32) << 16);
            const long long p = p0 + warp * 32 + lane;
            if (g.outTag == T_F16) {
                epilogue<__half, BN>(g, mine, p, q0, alpha);
            } else if (g.outTag == T_BF16) {
                epilogue<__nv_bfloat16, BN>(g, mine, p, q0, alpha);
            } else {
                epilogue<float, BN>(g, mine, p, q0, alpha);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 5) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(S::cols) : "memory");
    }
    if (threadIdx.x == 0 && *stalled) atomicCAS(g.err, E_NONE, E_STALLED);
}

// ---------------------------------------------------------------------------- host
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encodeTiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    if (!fn) throw CudaFail("the driver has no cuTensorMapEncodeTiled");
    return fn;
}

// Codes as a matrix of bytes; what lies behind its last row or column is read as 0, the code of 0.
CUtensorMap mapOf(const b200c_mx_matrix& m, int boxRows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(mxPitch(m.cols)), static_cast<cuuint64_t>(m.rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(m.ld)};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(boxRows)};
    const cuuint32_t step[2] = {1, 1};
    const CUresult r = encodeTiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m.codes, dims, strides, box, step,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw CudaFail("cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
    return map;
}

template <int BN, bool NV>
void launchTileOf(Context* ctx, const b200c_mx_matrix& p, const b200c_mx_matrix& q, MxMatmulParams g) {
    typedef Tile<BN, NV> S;
    static std::atomic<unsigned long long> ready{0};  // devices that have been told of the shared memory
    const unsigned long long bit = 1ull << (ctx->device & 63);
    if (!(ready.load() & bit)) {
        B2_CUDA(cudaFuncSetAttribute(mxMatmulKernel<BN, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smemBytes));
        ready.fetch_or(bit);
    }
    const CUtensorMap mapP = mapOf(p, 128), mapQ = mapOf(q, BN);
    g.tilesQ = static_cast<int>((q.rows + BN - 1) / BN);
    const long long tiles = (p.rows + 127) / 128 * g.tilesQ;
    if (tiles > 0x7FFFFFFFll) throw BadArg("the product has too many tiles");
    mxMatmulKernel<BN, NV><<<static_cast<unsigned int>(tiles), kThreads, S::smemBytes, ctx->stream>>>(mapP, mapQ, g);
    B2_CUDA(cudaGetLastError());
    ++ctx->launches;
}

template <int BN>
void launchFormat(Context* ctx, const b200c_mx_matrix& p, const b200c_mx_matrix& q, const MxMatmulParams& g) {
    if (p.format == B200C_NVFP4) {
        launchTileOf<BN, true>(ctx, p, q, g);
    } else {
        launchTileOf<BN, false>(ctx, p, q, g);
    }
}

}  // namespace

void launchMxMatmul(Context* ctx, const b200c_mx_matrix& a, const b200c_mx_matrix& b, void* out, int dtype, int64_t outLd) {
    if (a.rows == 0 || b.rows == 0) return;
    const int es = dtBits(dtype) / 8;
    if (a.cols == 0) {  // sums over nothing
        ++ctx->directOps;
        B2_CUDA(cudaMemset2DAsync(out, static_cast<size_t>(outLd * es), 0, static_cast<size_t>(b.rows * es), static_cast<size_t>(a.rows),
                                  ctx->stream));
        return;
    }
    // a side of up to 128 rows becomes the columns of a tile, which may be few
    const bool across = a.rows <= 128 && a.rows < b.rows;
    const b200c_mx_matrix& p = across ? b : a;
    const b200c_mx_matrix& q = across ? a : b;
    const bool nv = a.format == B200C_NVFP4;
    MxMatmulParams g;
    g.scalesP = static_cast<const unsigned char*>(p.scales);
    g.scalesQ = static_cast<const unsigned char*>(q.scales);
    g.tensorP = nv ? p.tensor_scale : nullptr;
    g.tensorQ = nv ? q.tensor_scale : nullptr;
    g.rowsP = p.rows;
    g.rowsQ = q.rows;
    g.k = a.cols;
    g.chunks = (mxBlocks(a.format, a.cols) + 3) / 4;
    g.scaleTilesQ = static_cast<int>((q.rows + 127) / 128);
    g.ktiles = static_cast<int>((a.cols + kTileK - 1) / kTileK);
    g.tilesQ = 0;
    g.out = out;
    g.ld = outLd;
    g.outTag = dtype == B200C_F16 ? T_F16 : dtype == B200C_BF16 ? T_BF16 : T_F32;
    g.across = across;
    g.wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (outLd * es) % 16 == 0;
    g.err = ctx->errWord;
    if (q.rows <= 16) {
        launchFormat<16>(ctx, p, q, g);
    } else if (q.rows <= 64) {
        launchFormat<64>(ctx, p, q, g);
    } else if (q.rows <= 128) {
        launchFormat<128>(ctx, p, q, g);
    } else {
        launchFormat<256>(ctx, p, q, g);
    }
}

}  // namespace b200c
