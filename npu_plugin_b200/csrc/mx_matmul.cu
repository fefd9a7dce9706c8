// Product of two block-scaled 4-bit matrices, out = A B^T, on the tensor cores (formats and storage:
// include/b200const.h).
//
// sum_k A[i][k] B[j][k] with A[i][k] = code * scale: tcgen05.mma takes the codes from shared memory and the
// scales from tensor memory and multiplies both in, 64 elements of k at a time; sums are 32 bits wide.
// One side's rows are the 128 rows of a tile ("P"), the other's its columns ("Q").
//
// Two kernels.  mxMatmulPairKernel, for products of many tiles, is bound by the tensor pipe, and by power where it
// runs long: 8192 x 4096 x 11008 (nvfp4) 125 us, 5.9 PFLOP/s -- 150 us in a long run, at 1000 W and 1.38 GHz.  Its tile of 256 x 256 for
// two SMs is what the way from L2 allows: an SM takes 64 bytes a clock, and a 128 x 256 tile of one SM would need
// 54 KB for 512 clocks of products, this one 38 KB.  mxMatmulKernel, for few rows on the left, is bound by that way from L2
// and by latency: 1 x 11008 x 4096 (nvfp4) 6.4 us, 16 x 4096 x 11008 (mxfp4) 6.4 us, and with weights from DRAM
// 1 x 32000 x 11008 30.8 us, 93 % of the copy rate.
#include "mx.h"
#include "runtime.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

namespace b200c {

namespace {

struct MxMatmulParams {
    const unsigned char* scalesP;
    const unsigned char* scalesQ;
    const float* tensorP;  // nvfp4
    const float* tensorQ;
    long long rowsP, rowsQ, k;
    long long chunks;      // tiles of 4 blocks along k: 512 bytes of scales each, per 128 rows
    int ktiles;
    int tilesP, tilesQ;
    int split;             // CTAs that share a tile's k
    void* out;
    long long ld;
    int outTag;            // T_F16, T_BF16, T_F32
    int wide;              // rows of the product are 16-byte aligned
    int bulkTo;            // column that bulk stores may reach: of rows that end inside a 16-byte line they would fill the line with zeros
    int* err;
};

constexpr int kTileK = 256;      // elements of k per stage: 128 bytes of codes, one swizzle row
constexpr int kStepK = 64;       // elements of k per tcgen05.mma
constexpr int kThreads = 192;    // warps 0-3: epilogue, 4: loads, 5: mma

// One CTA, 128 rows of P by BN rows of Q.
template <int BN, bool NV>
struct Tile {
    static constexpr int chunksPerTile = NV ? 4 : 2;  // 512-byte tiles of scales per stage and 128 rows
    static constexpr int bytesP = 128 * 128;
    static constexpr int bytesQ = BN * 128;
    static constexpr int scaleBytes = chunksPerTile * 512;  // of each side: a tile of Q begins where 128 rows do
    static constexpr int stageBytes = (bytesP + bytesQ + 2 * scaleBytes + 1023) / 1024 * 1024;
    // two CTAs fit an SM; more stages where one CTA has it to itself gained nothing
    static constexpr int stages = BN <= 16 ? 5 : BN <= 32 ? 4 : 3;
    static constexpr int smemBytes = 1024 /* alignment */ + stages * stageBytes;
    static constexpr int scaleCols = 2 * chunksPerTile * 4;  // tensor memory columns of a stage's scales
    static constexpr int scaleBufs = 2;
    static constexpr int needCols = BN + scaleBufs * scaleCols;
    static constexpr int cols = needCols <= 64 ? 64 : needCols <= 128 ? 128 : 256;
    static_assert(stages * stageBytes >= 128 * BN * 4, "the sums of a tile use the stages' memory on their way out");
};

// Two CTAs, 256 rows of P by 256 rows of Q: each CTA holds 128 rows of both sides and the sums of its 128
// rows of P.  Tensor memory: the sums of alternate tiles lie in columns 0..255 and 160..415, the scales behind.
template <bool NV>
struct PairTile {
    static constexpr int chunksPerTile = NV ? 4 : 2;
    static constexpr int bytesSide = 128 * 128;
    static constexpr int scaleBytes = chunksPerTile * 512;  // of 128 rows
    static constexpr int stageBytes = (2 * bytesSide + 3 * scaleBytes + 1023) / 1024 * 1024;
    static constexpr int stages = 5;
    static constexpr int stagingBytes = 2 * 32 * 128;  // of an epilogue warp: two groups of 32 x 32 values on their way out
    static constexpr int smemBytes = 1024 + stages * stageBytes + 4 * stagingBytes;
    static constexpr int accStep = 160, scaleCol = 416;
    static constexpr int scaleCols = 3 * chunksPerTile * 4;
    static constexpr int scaleBufs = 96 / scaleCols;
    static constexpr int cols = 512;
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

// The kernels here and those of mx_kernels.cu are launched so that the next one's CTAs may start while the last
// ones of this are at work (programmatic stream serialisation): nothing that another kernel wrote or reads is
// touched, and no tensor memory taken, before afterLast(); allowNext() comes behind the CTA's own allocation.
__device__ __forceinline__ void afterLast() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void allowNext() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void prefetchMap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// One thread of the warp, the same one every time and known to the compiler as such: the operands of
// what it issues stay in uniform registers.  Issued from a lane picked by its number the same
// instructions took 1.9 times as long (0.91 instead of 0.48 us per 256 elements of k of a 128 x 256 tile).
__device__ __forceinline__ bool electOne() {
    unsigned int one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ unsigned int clusterRank() {
    unsigned int r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void clusterSync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned int addrIn(unsigned int addr, unsigned int rank) {
    unsigned int r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void expectBytes(unsigned int bar, unsigned int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// After a wait that gave up: what was issued goes on all the same -- loads write shared memory, products read it and write
// tensor memory, commits arrive at barriers -- so a CTA frees and leaves nothing before all of it is done.  The barriers
// say when: use number n of a barrier completes its phase n.  These waits have the same limit.
__device__ __noinline__ void drain(unsigned int bar, int use) {
    const long long start = clock64();
    while (!barTry(bar, use & 1) && clock64() - start < 4000000000ll) {
    }
}
// the last use of each of a ring of barriers, `uses` in all
__device__ __noinline__ void drainRing(unsigned int bars, int stages, int uses) {
    for (int i = max(0, uses - stages); i < uses; ++i) drain(bars + 8 * (i % stages), i / stages);
}
__device__ __forceinline__ void storeIn(unsigned int addr, unsigned int rank, int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addrIn(addr, rank)), "r"(v) : "memory");
}
// `bytes` that will not come are counted as if they had
__device__ __forceinline__ void forgoBytes(unsigned int bar, unsigned int bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
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

// The same loads for one CTA of a pair, counted at a barrier of either.
__device__ __forceinline__ void loadTilePair(unsigned int dst, const CUtensorMap* map, int x, int y, unsigned int bar) {
    asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void loadScalesPair(unsigned int dst, const CUtensorMap* map, int chunk, int tile, unsigned int bar) {
    asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                    dst),
            "l"(map), "r"(0), "r"(chunk), "r"(tile), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void copyScalesPair(unsigned int tmem, unsigned long long desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

#define B2_MX_MMA(group, kind)                                                                                              \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::" group ".kind::" kind                  \
                 " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                                         \
                 "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate)                                      \
                 : "memory")
template <bool NV, bool PAIR>
__device__ __forceinline__ void mma(unsigned int d, unsigned long long a, unsigned long long b, unsigned int idesc,
                                    unsigned int scaleA, unsigned int scaleB, unsigned int accumulate) {
    if (NV && PAIR) {
        B2_MX_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    } else if (NV) {
        B2_MX_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    } else if (PAIR) {
        B2_MX_MMA("2", "mxf4.block_scale.scale_vec::2X");
    } else {
        B2_MX_MMA("1", "mxf4.block_scale.scale_vec::2X");
    }
}
#undef B2_MX_MMA
// arrives at `bar` (of both CTAs of a pair) once everything issued so far by this thread to the tensor core is done
__device__ __forceinline__ void mmaCommit(unsigned int bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mmaCommitPair(unsigned int bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<unsigned short>(3))
                 : "memory");
}

// Instruction descriptor: e2m1 x e2m1, M x N; the scales' type in bit 23 (1: e8m0); which pair of a word's
// four scale bytes is meant in bits 29 (A) and 4 (B).
template <int M, int N, bool NV>
__device__ __forceinline__ unsigned int instruction(int pair) {
    return (1u << 7) | (1u << 10) | (static_cast<unsigned int>(N >> 3) << 17) | (NV ? 0u : 1u << 23) |
           (static_cast<unsigned int>(M >> 7) << 27) | (static_cast<unsigned int>(pair) << 29) | (static_cast<unsigned int>(pair) << 4);
}

// The products of one stage: up to four steps of 64 elements of k.  A word of four scales reaches over one step
// (nvfp4) or two (mxfp4); `wordsQ` columns of tensor memory lie between the words of Q.
template <int M, int N, bool NV, bool PAIR>
__device__ __forceinline__ void mmaStage(unsigned int acc, unsigned long long dp, unsigned long long dq, unsigned int colP,
                                         unsigned int colQ, int wordsQ, int steps, bool first) {
#pragma unroll
    for (int i = 0; i < kTileK / kStepK; ++i) {
        if (i < steps) {
            const int c = NV ? i : i >> 1, pair = NV ? 0 : (i & 1) * 2;
            mma<NV, PAIR>(acc, dp + i * 2, dq + i * 2, instruction<M, N, NV>(pair), colP + c * 4, colQ + c * wordsQ, !(first && i == 0));
        }
    }
}

// 32 columns of this warp's lanes; the values are there after readsDone()
__device__ __forceinline__ void startRead(unsigned int addr, unsigned int r[32]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
              "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
              "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(addr)
            : "memory");
}
// ties the registers of a read to the wait, so that nothing uses them before it
__device__ __forceinline__ void readsDone(unsigned int r[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
    asm volatile(""
                 : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void readColumns(unsigned int addr, float v[32]) {
    unsigned int r[32];
    startRead(addr, r);
    readsDone(r);
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

// What a sum is multiplied with, one factor after the other.  Where the product of the tensor scales is a normal number
// it is the first, and the second is 1.  Otherwise that product would lose what the result still has -- two matrices
// of size 2^-64 have scales around 2^-75, whose product 32 bits do not hold -- or be an infinity that makes NaN of a sum of
// zeros.  Sums are 0 or lie within 2^-20 .. 2^54 (codes of 0.5 with scales of 2^-9 on both sides; 36 * 448^2 for each
// of 2^31 elements), so the exponent is shared out evenly: a product with the first factor is below the normal numbers
// only where the result is 0 anyway, and above the largest only where the result is, too.
template <bool NV>
struct Factors {};  // mxfp4 has none
template <>
struct Factors<true> {
    float first, second;
};
__device__ __noinline__ Factors<true> farFactors(float tp, float tq) {
    int ep, eq;
    const float m = frexpf(tp, &ep) * frexpf(tq, &eq);
    // beyond these the result is 0 or infinity whatever the sum
    const int e = min(max(ep + eq, -212), 200);
    return Factors<true>{ldexpf(m, e / 2), ldexpf(1.f, e - e / 2)};
}
template <bool NV>
__device__ __forceinline__ Factors<NV> factorsOf(const MxMatmulParams&) {
    return {};
}
template <>
__device__ __forceinline__ Factors<true> factorsOf<true>(const MxMatmulParams& g) {
    const float tp = g.tensorP[0], tq = g.tensorQ[0], product = tp * tq;
    const bool normal = fabsf(product) >= 1.17549435e-38f && fabsf(product) <= 3.402823466e38f;
    // a scale that is 0, infinite or NaN has only the product that it has
    if (normal || tp == 0.f || tq == 0.f || !(fabsf(tp) <= 3.402823466e38f && fabsf(tq) <= 3.402823466e38f)) return {product, 1.f};
    return farFactors(tp, tq);
}

// N sums times both factors, two at a time
template <int N>
__device__ __forceinline__ void scaled(const Factors<false>&, float*) {
}
template <int N>
__device__ __forceinline__ void scaled(const Factors<true>& f, float* v) {
    static_assert(N % 2 == 0, "pairs");
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        asm("{\n\t.reg .b64 v, a, b;\n\t"
            "mov.b64 v, {%0, %1};\n\tmov.b64 a, {%2, %2};\n\tmov.b64 b, {%3, %3};\n\t"
            "mul.rn.f32x2 v, v, a;\n\tmul.rn.f32x2 v, v, b;\n\t"
            "mov.b64 {%0, %1}, v;\n\t}"
            : "+f"(v[i]), "+f"(v[i + 1])
            : "f"(f.first), "f"(f.second));
    }
}

// The single-CTA kernel's P is the right matrix: N accumulator columns of lane p are N rows of the product at
// column p, and a warp's lanes store 32 neighbours at a time.
template <class T, int N>
__device__ __forceinline__ void storeAcross(const MxMatmulParams& g, long long p, long long q0, const float* v) {
    if (p >= g.rowsP) return;
    const long long left = g.rowsQ - q0;
    T* at = static_cast<T*>(g.out) + q0 * g.ld + p;
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; ++i, at += g.ld) *at = toOut<T>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i, at += g.ld)
            if (i < left) *at = toOut<T>(v[i]);
    }
}
template <class T, int BN, bool NV>
__device__ __forceinline__ void epilogue(const MxMatmulParams& g, unsigned int acc, long long p, long long q0, const Factors<NV>& f) {
    constexpr int n = BN < 32 ? BN : 32;
#pragma unroll 1
    for (int c = 0; c < BN && q0 + c < g.rowsQ; c += n) {
        float v[32];
        if (n == 32) {
            readColumns(acc + c, v);
        } else {
            readColumns16(acc + c, v);
        }
        scaled<n>(f, v);
        storeAcross<T, n>(g, p, q0 + c, v);
    }
}

// A tile whose k is shared out: its sums lie in `split` (at most MOST) CTAs' shared memory as [BN][128]; this CTA adds
// up its share of the columns, in the order of the ranks, so that the result is the same on every run.  A thread takes
// four rows at a time, and 16 loads from the cluster's memory are under way at once: with one column at a time the
// waiting for them took longer than the product itself.
template <class T, int BN, int MOST, bool NV>
__device__ __forceinline__ void joinColumns(const MxMatmulParams& g, unsigned int sums, unsigned int rank, int thread, long long p0,
                                            long long q0, const Factors<NV>& f) {
    constexpr int most = 16 / MOST;
    const int c0 = static_cast<int>(rank) * BN / g.split, c1 = (static_cast<int>(rank) + 1) * BN / g.split;
    const int row = thread % 32 * 4;
    const long long p = p0 + row;
    const int rows = static_cast<int>(min(4ll, g.rowsP - p)), cols = static_cast<int>(min(static_cast<long long>(c1), g.rowsQ - q0));
    if (rows <= 0) return;
    unsigned int from[MOST];
#pragma unroll
    for (int r = 0; r < MOST; ++r) from[r] = addrIn(sums + row * 4, min(r, g.split - 1));
    for (int c = c0 + thread / 32; c < cols; c += 4 * most) {
        float w[most][MOST][4];
#pragma unroll
        for (int j = 0; j < most; ++j) {
#pragma unroll
            for (int r = 0; r < MOST; ++r) {
                if (r < g.split && c + 4 * j < cols) {
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(w[j][r][0]), "=f"(w[j][r][1]), "=f"(w[j][r][2]), "=f"(w[j][r][3])
                                 : "r"(from[r] + (c + 4 * j) * 512)
                                 : "memory");
                }
            }
        }
#pragma unroll
        for (int j = 0; j < most; ++j) {
            const long long q = q0 + c + 4 * j;
            if (c + 4 * j >= cols) break;
            alignas(16) T v[4];
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = w[j][0][i];
#pragma unroll
                for (int r = 1; r < MOST; ++r)
                    if (r < g.split) s[i] = s[i] + w[j][r][i];
            }
            scaled<4>(f, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = toOut<T>(s[i]);
            T* out = static_cast<T*>(g.out);
            if (g.wide && rows == 4) {
                T* at = out + q * g.ld + p;
                if (sizeof(T) == 4) {
                    *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(v);
                } else {
                    *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(v);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < rows) out[q * g.ld + p + i] = v[i];
            }
        }
    }
}

template <class T, int BN, bool NV>
__device__ __forceinline__ void join(const MxMatmulParams& g, unsigned int sums, unsigned int rank, int thread, long long p0, long long q0,
                                     const Factors<NV>& f) {
    if (g.split <= 2) {
        joinColumns<T, BN, 2, NV>(g, sums, rank, thread, p0, q0, f);
    } else if (g.split <= 4) {
        joinColumns<T, BN, 4, NV>(g, sums, rank, thread, p0, q0, f);
    } else {
        joinColumns<T, BN, 8, NV>(g, sums, rank, thread, p0, q0, f);
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
    constexpr int stages = S::stages;
    const unsigned int full = smemAddr(bars), empty = full + 8 * S::stages, done = empty + 8 * S::stages;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned int rank = g.split > 1 ? clusterRank() : 0;
    const int tile = blockIdx.x / g.split;
    const long long p0 = static_cast<long long>(tile / g.tilesQ) * 128;
    const long long q0 = static_cast<long long>(tile % g.tilesQ) * BN;
    const int k0 = static_cast<int>(static_cast<long long>(g.ktiles) * rank / g.split);
    const int n = static_cast<int>(static_cast<long long>(g.ktiles) * (rank + 1) / g.split) - k0;

    if (threadIdx.x == 0) {
        prefetchMap(&mapP);
        prefetchMap(&mapQ);
        for (int s = 0; s < stages; ++s) {
            barInit(full + 8 * s, 1);
            barInit(empty + 8 * s, 1);
        }
        barInit(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        stalledWord = 0;
    }
    afterLast();
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemBase)), "r"(S::cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    allowNext();
    const unsigned int acc = tmemBase, scaleCol = tmemBase + BN;
    int issued = 0;  // stages whose loads (warp 4) or products (warp 5) have been issued

    if (warp == 4) {
        const long long scaleTileP = p0 / 128, scaleTileQ = q0 / 128;
        int s = 0, phase = 1;
        for (; issued < n; ++issued) {
            if (!__all_sync(0xFFFFFFFFu, issued < stages || barWait(empty + 8 * s, phase, stalled))) break;
            if (electOne()) {
                const int kt = k0 + issued;
                const unsigned int at = stage0 + s * S::stageBytes, bar = full + 8 * s;
                const long long chunk = static_cast<long long>(kt) * S::chunksPerTile;
                const unsigned int scaleBytes = static_cast<unsigned int>(min(static_cast<long long>(S::chunksPerTile), g.chunks - chunk)) * 512u;
                expectBytes(bar, S::bytesP + S::bytesQ + 2 * scaleBytes);
                loadTile(at, &mapP, kt * 128, static_cast<int>(p0), bar);
                loadTile(at + S::bytesP, &mapQ, kt * 128, static_cast<int>(q0), bar);
                const unsigned int sp = at + S::bytesP + S::bytesQ;
                loadBytes(sp, g.scalesP + (scaleTileP * g.chunks + chunk) * 512, scaleBytes, bar);
                loadBytes(sp + S::scaleBytes, g.scalesQ + (scaleTileQ * g.chunks + chunk) * 512, scaleBytes, bar);
            }
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1;
        }
    } else if (warp == 5) {
        const unsigned long long dp0 = operandDesc(stage0), dq0 = operandDesc(stage0 + S::bytesP);
        const unsigned long long ds0 = scaleDesc(stage0 + S::bytesP + S::bytesQ);
        int s = 0, phase = 0, before = 0, beforePhase = 0;  // before: the stage scaleBufs ago
        for (int i = 0; i < n; ++i, ++issued) {
            if (!__all_sync(0xFFFFFFFFu, barWait(full + 8 * s, phase, stalled))) break;
            // the scales' columns are free once the products that read them are done: nothing else orders a copy behind them
            if (i >= S::scaleBufs) {
                if (!__all_sync(0xFFFFFFFFu, barWait(empty + 8 * before, beforePhase, stalled))) break;
                if (++before == stages) before = 0, beforePhase ^= 1;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (electOne()) {
                const int kt = k0 + i;
                const unsigned int colP = scaleCol + (i % S::scaleBufs) * S::scaleCols, colQ = colP + S::chunksPerTile * 4;
                const unsigned long long off = static_cast<unsigned long long>(s * (S::stageBytes >> 4));
                if (kt + 1 < g.ktiles) {
#pragma unroll
                    for (int c = 0; c < S::chunksPerTile; ++c) {
                        copyScales(colP + c * 4, ds0 + off + c * 32);
                        copyScales(colQ + c * 4, ds0 + off + S::scaleBytes / 16 + c * 32);
                    }
                    mmaStage<128, BN, NV, false>(acc, dp0 + off, dq0 + off, colP, colQ, 4, kTileK / kStepK, i == 0);
                } else {  // the last of k: what scales there are
                    const int chunks = static_cast<int>(g.chunks - static_cast<long long>(kt) * S::chunksPerTile);
                    const int steps = static_cast<int>((g.k - static_cast<long long>(kt) * kTileK + kStepK - 1) / kStepK);
#pragma unroll
                    for (int c = 0; c < S::chunksPerTile; ++c) {
                        if (c < chunks) {
                            copyScales(colP + c * 4, ds0 + off + c * 32);
                            copyScales(colQ + c * 4, ds0 + off + S::scaleBytes / 16 + c * 32);
                        }
                    }
                    mmaStage<128, BN, NV, false>(acc, dp0 + off, dq0 + off, colP, colQ, 4, steps, i == 0);
                }
                mmaCommit(empty + 8 * s);
                if (i + 1 == n) mmaCommit(done);
            }
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1;
        }
    }
    __syncwarp();
    const Factors<NV> f = factorsOf<NV>(g);  // before the wait, which hides its loads
    const bool finished = warp < 4 && __all_sync(0xFFFFFFFFu, barWait(done, 0, stalled) && !*stalled);  // the reads are the whole warp's
    const unsigned int mine = acc + (static_cast<unsigned int>(warp * 32) << 16);
    const int row = warp * 32 + lane;
    if (finished) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (g.split == 1) {
        if (finished) {
            if (g.outTag == T_F16) {
                epilogue<__half, BN, NV>(g, mine, p0 + row, q0, f);
            } else if (g.outTag == T_BF16) {
                epilogue<__nv_bfloat16, BN, NV>(g, mine, p0 + row, q0, f);
            } else {
                epilogue<float, BN, NV>(g, mine, p0 + row, q0, f);
            }
        }
    } else {
        if (finished) {  // all products are done with the stages
            constexpr int w = BN < 32 ? BN : 32;
#pragma unroll 1
            for (int c = 0; c < BN && q0 + c < g.rowsQ; c += w) {
                float v[32];
                if (w == 32) {
                    readColumns(mine + c, v);
                } else {
                    readColumns16(mine + c, v);
                }
#pragma unroll
                for (int i = 0; i < w; ++i) {
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(stage0 + ((c + i) * 128 + row) * 4), "f"(v[i]) : "memory");
                }
            }
        }
        __syncwarp();
        clusterSync();
        if (finished) {
            if (g.outTag == T_F16) {
                join<__half, BN, NV>(g, stage0, rank, row, p0, q0, f);
            } else if (g.outTag == T_BF16) {
                join<__nv_bfloat16, BN, NV>(g, stage0, rank, row, p0, q0, f);
            } else {
                join<float, BN, NV>(g, stage0, rank, row, p0, q0, f);
            }
        }
        __syncwarp();
        clusterSync();  // the others have read this CTA's sums
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*stalled) {  // all warps see the same: none sets it behind the barrier
        if (warp == 4) drainRing(full, stages, issued);
        if (warp == 5) {
            drainRing(empty, stages, issued);
            if (issued == n) drain(done, 0);
        }
        __syncthreads();
    }
    if (warp == 5) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(S::cols) : "memory");
    }
    if (threadIdx.x == 0 && *stalled) atomicCAS(g.err, E_NONE, E_STALLED);
}

// Tile t of the sweep: eight tiles of P down, then on to the next of Q, so that the tiles in flight form a
// block and share their operands in L2.
__device__ __forceinline__ void tileOf(const MxMatmulParams& g, int t, int* p, int* q) {
    constexpr int G = 8;
    const int group = t / (G * g.tilesQ), r = t - group * G * g.tilesQ;
    const int high = min(G, g.tilesP - group * G);
    *q = r / high;
    *p = group * G + (r - *q * high);
}

// 32 columns of a warp's 32 rows, staged as storeGroup() lays them, in rows that no bulk store can start at or end in: the
// warp stores them one by one, 32 neighbours at a time.
template <class T>
__device__ __forceinline__ void storeRows(const MxMatmulParams& g, unsigned int at, int lane, long long row0, long long col0) {
    constexpr int rowBytes = 32 * sizeof(T), chunks = rowBytes / 16;
    const int rows = static_cast<int>(min(32ll, g.rowsP - row0));
    T* out = static_cast<T*>(g.out) + row0 * g.ld + col0 + lane;
    const bool mine = col0 + lane < g.rowsQ;
    const int c = lane * static_cast<int>(sizeof(T)) / 16, in = lane * static_cast<int>(sizeof(T)) % 16;
#pragma unroll 8
    for (int i = 0; i < 32; ++i, out += g.ld) {
        if (i < rows && mine) {
            const unsigned int from = at + i * rowBytes + ((c ^ (chunks == 8 ? i & 7 : (i >> 1) & 3)) << 4) + in;
            if (sizeof(T) == 2) {
                unsigned short w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(from) : "memory");
                *reinterpret_cast<unsigned short*>(out) = w;
            } else {
                unsigned int w;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(from) : "memory");
                *reinterpret_cast<unsigned int*>(out) = w;
            }
        }
    }
}
// 32 columns of a warp's 32 rows -> the product, through shared memory and a bulk store: a row's 32 values are
// 64 or 128 bytes, which leave together, where a thread's own stores of its row would be 16 bytes of 32
// different rows at a time.
template <class T, bool NV>
__device__ __forceinline__ void storeGroup(const MxMatmulParams& g, const CUtensorMap* mapOut, unsigned int staging, int group, int lane,
                                           long long row0, long long col0, const unsigned int r[32], const Factors<NV>& f) {
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
    scaled<32>(f, v);
    constexpr int rowBytes = 32 * sizeof(T), chunks = rowBytes / 16, bufs = 2 * 128 / rowBytes;
    const unsigned int at = staging + (group % bufs) * 32 * rowBytes;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(bufs - 1) : "memory");  // the last store from here has been read
    __syncwarp();
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
        alignas(16) T t[16 / sizeof(T)];
#pragma unroll
        for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) t[j] = toOut<T>(v[c * (16 / sizeof(T)) + j]);
        const uint4 w = *reinterpret_cast<const uint4*>(t);
        // the map's swizzle: 16-byte chunks of a row of 64 or 128 bytes change places with the row's number
        const unsigned int to = at + lane * rowBytes + ((c ^ (chunks == 8 ? lane & 7 : (lane >> 1) & 3)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
    }
    if (!g.wide) {
        __syncwarp();
        storeRows<T>(g, at, lane, row0, col0);
        __syncwarp();
        return;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    const bool ends = col0 + 32 > g.bulkTo;  // inside a line
    if (ends) {
        storeRows<T>(g, at, lane, row0, col0);
        __syncwarp();
    }
    if (lane == 0) {
        if (row0 < g.rowsP && col0 < g.rowsQ && !ends) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(mapOut),
                         "r"(static_cast<int>(col0)), "r"(static_cast<int>(row0)), "r"(at)
                         : "memory");
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

template <class T, bool NV>
__device__ __forceinline__ void pairEpilogue(const MxMatmulParams& g, const CUtensorMap* mapOut, unsigned int staging, unsigned int acc, int buf,
                                             long long row0, long long q0, const Factors<NV>& f, unsigned int accFree, int lane) {
    // columns 160..255 of tensor memory belong to both buffers: they are read first, and the next tile may start
    const int shared0 = buf ? 0 : 160;
    unsigned int r[3][32];
#pragma unroll
    for (int i = 0; i < 3; ++i) startRead(acc + shared0 + i * 32, r[i]);
#pragma unroll
    for (int i = 0; i < 3; ++i) readsDone(r[i]);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(accFree) : "memory");
#pragma unroll
    for (int i = 0; i < 3; ++i) storeGroup<T, NV>(g, mapOut, staging, i, lane, row0, q0 + shared0 + i * 32, r[i], f);
    const int rest = buf ? 96 : 0;
#pragma unroll 1
    for (int i = 0; i < 5; ++i) {
        startRead(acc + rest + i * 32, r[0]);
        readsDone(r[0]);
        storeGroup<T, NV>(g, mapOut, staging, i + 3, lane, row0, q0 + rest + i * 32, r[0], f);
    }
}

template <bool NV>
__global__ void __launch_bounds__(kThreads) mxMatmulPairKernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
                                                               const __grid_constant__ CUtensorMap mapScalesP,
                                                               const __grid_constant__ CUtensorMap mapScalesQ,
                                                               const __grid_constant__ CUtensorMap mapOut,
                                                               const __grid_constant__ MxMatmulParams g) {
    typedef PairTile<NV> S;
    extern __shared__ unsigned char raw[];
    __shared__ unsigned long long bars[2 * S::stages + 2];
    __shared__ unsigned int tmemBase;
    __shared__ int stalledWord, peerStalled;
    __shared__ int loadsOf[2], productsDone, tilesDone;  // of each CTA's loads, and of the first CTA's products: stages issued
    volatile int* stalled = &stalledWord;
    const unsigned int stage0 = (smemAddr(raw) + 1023u) & ~1023u;
    const unsigned int full = smemAddr(bars), empty = full + 8 * S::stages, accFull = empty + 8 * S::stages, accFree = accFull + 8;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned int rank = clusterRank();
    const int tiles = g.tilesP * g.tilesQ, pairs = gridDim.x / 2;

    if (threadIdx.x == 0) {
        prefetchMap(&mapP);
        prefetchMap(&mapQ);
        prefetchMap(&mapScalesP);
        prefetchMap(&mapScalesQ);
        if (g.wide) prefetchMap(&mapOut);
        for (int s = 0; s < S::stages; ++s) {
            barInit(full + 8 * s, 1);
            barInit(empty + 8 * s, 1);
        }
        barInit(accFull, 1);
        barInit(accFree, 8);  // four epilogue warps of both CTAs
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        stalledWord = peerStalled = 0;
    }
    afterLast();
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemBase)), "r"(S::cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    clusterSync();  // both CTAs' barriers are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    allowNext();
    const unsigned int tmem = tmemBase;

    if (warp == 4) {
        // each CTA loads its halves; what they bring is counted at the first CTA's barrier, where the products wait
        const unsigned int full0 = addrIn(full, 0);
        int s = 0, phase = 1, issued = 0;
        bool ok = true;
        for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs) {
            int tp, tq;
            tileOf(g, t, &tp, &tq);
            for (int kt = 0; kt < g.ktiles; ++kt, ++issued) {
                ok = __all_sync(0xFFFFFFFFu, issued < S::stages || barWait(empty + 8 * s, phase, stalled));
                if (!ok) break;
                if (electOne()) {
                    const unsigned int at = stage0 + s * S::stageBytes, bar = full0 + 8 * s;
                    if (rank == 0) expectBytes(full + 8 * s, 2 * (2 * S::bytesSide + 3 * S::scaleBytes));
                    loadTilePair(at, &mapP, kt * 128, tp * 256 + static_cast<int>(rank) * 128, bar);
                    loadTilePair(at + S::bytesSide, &mapQ, kt * 128, tq * 256 + static_cast<int>(rank) * 128, bar);
                    const unsigned int sp = at + 2 * S::bytesSide;
                    loadScalesPair(sp, &mapScalesP, kt * S::chunksPerTile, tp * 2 + static_cast<int>(rank), bar);
                    loadScalesPair(sp + S::scaleBytes, &mapScalesQ, kt * S::chunksPerTile, tq * 2, bar);
                }
                __syncwarp();
                if (++s == S::stages) s = 0, phase ^= 1;
            }
        }
        if (lane < 2) storeIn(smemAddr(&loadsOf[rank]), lane, issued);
    } else if (warp == 5 && rank == 0) {
        const unsigned long long dp0 = operandDesc(stage0), dq0 = operandDesc(stage0 + S::bytesSide);
        const unsigned long long ds0 = scaleDesc(stage0 + 2 * S::bytesSide);
        int s = 0, phase = 0, it = 0, done = 0;
        int before = 0, beforePhase = 0;  // the stage, scaleBufs ago, whose products must be done with their scales
        int whole = 0;  // tiles whose products have all been issued
        bool ok = true;
        for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs, ++done) {
            const unsigned int acc = tmem + (done & 1) * S::accStep;
            if (done > 0) ok = __all_sync(0xFFFFFFFFu, barWait(accFree, (done - 1) & 1, stalled));
            for (int kt = 0; kt < g.ktiles && ok; ++kt, ++it) {
                ok = barWait(full + 8 * s, phase, stalled);
                // as above: a copy of scales waits for the products that read the columns before
                if (it >= S::scaleBufs) {
                    ok = ok && barWait(empty + 8 * before, beforePhase, stalled);
                    if (++before == S::stages) before = 0, beforePhase ^= 1;
                }
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (electOne()) {
                    const unsigned int colP = tmem + S::scaleCol + (it % S::scaleBufs) * S::scaleCols, colQ = colP + S::chunksPerTile * 4;
                    const unsigned long long off = static_cast<unsigned long long>(s * (S::stageBytes >> 4));
#pragma unroll
                    for (int c = 0; c < S::chunksPerTile; ++c) {
                        copyScalesPair(colP + c * 4, ds0 + off + c * 32);
                        copyScalesPair(colQ + c * 8, ds0 + off + S::scaleBytes / 16 + c * 32);
                        copyScalesPair(colQ + c * 8 + 4, ds0 + off + S::scaleBytes / 8 + c * 32);
                    }
                    if (kt + 1 < g.ktiles) {
                        mmaStage<256, 256, NV, true>(acc, dp0 + off, dq0 + off, colP, colQ, 8, kTileK / kStepK, kt == 0);
                    } else {
                        const int steps = static_cast<int>((g.k - static_cast<long long>(kt) * kTileK + kStepK - 1) / kStepK);
                        mmaStage<256, 256, NV, true>(acc, dp0 + off, dq0 + off, colP, colQ, 8, steps, kt == 0);
                    }
                    mmaCommitPair(empty + 8 * s);
                    if (kt + 1 == g.ktiles) mmaCommitPair(accFull);
                }
                __syncwarp();
                if (++s == S::stages) s = 0, phase ^= 1;
                if (kt + 1 == g.ktiles) ++whole;
            }
        }
        if (lane < 2) {
            storeIn(smemAddr(&productsDone), lane, it);
            storeIn(smemAddr(&tilesDone), lane, whole);
        }
    } else if (warp < 4) {
        const Factors<NV> f = factorsOf<NV>(g);
        const unsigned int accFree0 = addrIn(accFree, 0);
        const unsigned int staging = stage0 + S::stages * S::stageBytes + warp * S::stagingBytes;
        int done = 0;
        for (int t = blockIdx.x / 2; t < tiles; t += pairs, ++done) {
            int tp, tq;
            tileOf(g, t, &tp, &tq);
            if (!__all_sync(0xFFFFFFFFu, barWait(accFull, done & 1, stalled) && !*stalled)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int buf = done & 1;
            const unsigned int acc = tmem + buf * S::accStep + (static_cast<unsigned int>(warp * 32) << 16);
            const long long row0 = static_cast<long long>(tp) * 256 + rank * 128 + warp * 32, q0 = static_cast<long long>(tq) * 256;
            if (g.outTag == T_F16) {
                pairEpilogue<__half, NV>(g, &mapOut, staging, acc, buf, row0, q0, f, accFree0, lane);
            } else if (g.outTag == T_BF16) {
                pairEpilogue<__nv_bfloat16, NV>(g, &mapOut, staging, acc, buf, row0, q0, f, accFree0, lane);
            } else {
                pairEpilogue<float, NV>(g, &mapOut, staging, acc, buf, row0, q0, f, accFree0, lane);
            }
        }
    }
    if (warp < 4 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the last stores are through
    __syncwarp();
    if (*stalled && lane == 0) storeIn(smemAddr(&peerStalled), rank ^ 1, 1);
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    clusterSync();  // neither CTA leaves while the other's products, copies or arrivals reach into it
    if (*stalled || *const_cast<volatile int*>(&peerStalled)) {  // both CTAs see the same
        if (warp == 4 && rank == 0) {
            // the loads of both CTAs are counted here; one of them may have gone on for some stages
            constexpr unsigned int half = 2 * S::bytesSide + 3 * S::scaleBytes;
            const int n0 = loadsOf[0], n1 = loadsOf[1];
            drainRing(full, S::stages, min(n0, n1));
            for (int i = min(n0, n1); i < max(n0, n1); ++i) {
                const unsigned int bar = full + 8 * (i % S::stages);
                if (lane == 0) {
                    if (n1 > n0) {
                        expectBytes(bar, half);
                    } else {
                        forgoBytes(bar, half);
                    }
                }
                __syncwarp();
                drain(bar, i / S::stages);
            }
        }
        if (warp == 5) {
            drainRing(empty, S::stages, productsDone);
            if (tilesDone > 0) drain(accFull, tilesDone - 1);
        }
        __syncwarp();
        clusterSync();
    }
    if (warp == 5) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(S::cols) : "memory");
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

// Scales as [row tiles][block tiles][512 bytes]; what lies behind either end is read as 0.
CUtensorMap scaleMapOf(const b200c_mx_matrix& m, int chunksPerTile, int boxTiles) {
    CUtensorMap map;
    const cuuint64_t chunks = static_cast<cuuint64_t>((mxBlocks(m.format, m.cols) + 3) / 4);
    const cuuint64_t dims[3] = {256, chunks, static_cast<cuuint64_t>((m.rows + 127) / 128)};
    const cuuint64_t strides[2] = {512, chunks * 512};
    const cuuint32_t box[3] = {256, static_cast<cuuint32_t>(chunksPerTile), static_cast<cuuint32_t>(boxTiles)};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = encodeTiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, m.scales, dims, strides, box, step,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw CudaFail("cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
    return map;
}

// The product as groups of 32 x 32 values; what lies behind its last row is not written, and behind its last column
// nothing beyond that one's 16 bytes, which a bulk store fills up with zeros: MxMatmulParams::bulkTo keeps it from there.
CUtensorMap outMapOf(void* out, int dtype, int64_t rows, int64_t cols, int64_t ld) {
    CUtensorMap map;
    const int es = dtBits(dtype) / 8;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * es)};
    const cuuint32_t box[2] = {32, 32};
    const cuuint32_t step[2] = {1, 1};
    const CUtensorMapDataType type = dtype == B200C_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : dtype == B200C_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    const CUresult r = encodeTiled()(&map, type, 2, out, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw CudaFail("cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
    return map;
}

// The kernel may use `bytes` of shared memory; told once per device.
template <class Kernel>
void allowSmem(Context* ctx, Kernel kernel, int bytes, std::atomic<unsigned long long>& ready) {
    const unsigned long long bit = 1ull << (ctx->device & 63);
    if (ready.load() & bit) return;
    B2_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    ready.fetch_or(bit);
}

template <class... Args>
void launchClusters(Context* ctx, void (*kernel)(Args...), unsigned int ctas, unsigned int perCluster, int smem,
                    typename std::common_type<Args>::type... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = perCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = perCluster > 1 ? 2 : 1;
    B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    ++ctx->launches;
}

// How many CTAs share a tile's k.  In us: a stage takes about 0.34 where its loads are waited for, the CTAs that do
// not fit the SMs one by one follow or share an SM, and joining the sums costs more the more there are of
// them.  Measured for 1 x 11008 x 4096 with 1, 2, 3, 4 CTAs: 7.6, 7.2, 6.6, 9.4; 16 x 4096 x 11008 with 1, 2, 4, 8:
// 15.7, 10.1, 6.6, 7.2; 128 x 4096 x 4096: 8.8, 8.2, 7.2, 10.2; 77 x 515 x 1003: 4.7, 6.3, 5.5.
int splitOf(Context* ctx, long long tiles, int ktiles, int bn) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 8 && s <= ktiles; ++s) {
        const long long rounds = (tiles * s + ctx->smCount - 1) / ctx->smCount;
        if (s > 1 && rounds > (bn <= 32 ? 2 : 1)) break;
        const double cost = 0.34 * static_cast<double>(rounds * ((ktiles + s - 1) / s)) * (rounds > 1 ? 0.9 : 1.0) +
                            (s > 1 ? 0.3 + 0.011 * bn + 0.05 * s : 0.0);
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

template <int BN, bool NV>
void launchTileOf(Context* ctx, const b200c_mx_matrix& p, const b200c_mx_matrix& q, MxMatmulParams g) {
    typedef Tile<BN, NV> S;
    static std::atomic<unsigned long long> ready{0};
    allowSmem(ctx, mxMatmulKernel<BN, NV>, S::smemBytes, ready);
    g.tilesP = static_cast<int>((p.rows + 127) / 128);
    g.tilesQ = static_cast<int>((q.rows + BN - 1) / BN);
    const long long tiles = static_cast<long long>(g.tilesP) * g.tilesQ;
    g.split = splitOf(ctx, tiles, g.ktiles, BN);
    if (tiles * g.split > 0x7FFFFFFFll) throw BadArg("the product has too many tiles");
    launchClusters(ctx, mxMatmulKernel<BN, NV>, static_cast<unsigned int>(tiles * g.split), static_cast<unsigned int>(g.split),
                   S::smemBytes, mapOf(p, 128), mapOf(q, BN), g);
}

template <bool NV>
void launchPairs(Context* ctx, const b200c_mx_matrix& p, const b200c_mx_matrix& q, int dtype, MxMatmulParams g) {
    typedef PairTile<NV> S;
    static std::atomic<unsigned long long> ready{0};
    allowSmem(ctx, mxMatmulPairKernel<NV>, S::smemBytes, ready);
    g.tilesP = static_cast<int>((p.rows + 255) / 256);
    g.tilesQ = static_cast<int>((q.rows + 255) / 256);
    const long long tiles = static_cast<long long>(g.tilesP) * g.tilesQ;
    if (tiles > 0x3FFFFFFFll) throw BadArg("the product has too many tiles");
    const long long pairs = std::min<long long>(tiles, ctx->smCount / 2);
    launchClusters(ctx, mxMatmulPairKernel<NV>, static_cast<unsigned int>(2 * pairs), 2u, S::smemBytes, mapOf(p, 128), mapOf(q, 128),
                   scaleMapOf(p, S::chunksPerTile, 1), scaleMapOf(q, S::chunksPerTile, 2),
                   g.wide ? outMapOf(g.out, dtype, p.rows, q.rows, g.ld) : CUtensorMap{}, g);
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
    // pairs from a quarter of the SMs in tiles on: 512 x 4096 x 4096 (32 tiles) takes 8.8 us by single CTAs and 9.9 by
    // pairs, 768 (48 tiles) 10.9 and 10.4
    const long long big = ((a.rows + 255) / 256) * ((b.rows + 255) / 256);
    const bool pairs = big >= ctx->smCount / 4 && a.rows > 128 && b.rows > 128;
    const b200c_mx_matrix& p = pairs ? a : b;
    const b200c_mx_matrix& q = pairs ? b : a;
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
    g.ktiles = static_cast<int>((a.cols + kTileK - 1) / kTileK);
    g.tilesP = g.tilesQ = 0;
    g.split = 1;
    g.out = out;
    g.ld = outLd;
    g.outTag = dtype == B200C_F16 ? T_F16 : dtype == B200C_BF16 ? T_BF16 : T_F32;
    g.wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (outLd * es) % 16 == 0 && outLd * es < (int64_t(1) << 40);
    g.bulkTo = q.rows * es % 16 != 0 ? static_cast<int>(q.rows) : 0x7FFFFFFF;
    g.err = ctx->errWord;
    if (pairs) {
        if (nv) {
            launchPairs<true>(ctx, p, q, dtype, g);
        } else {
            launchPairs<false>(ctx, p, q, dtype, g);
        }
    } else if (q.rows <= 16) {
        launchFormat<16>(ctx, p, q, g);
    } else if (q.rows <= 32) {
        launchFormat<32>(ctx, p, q, g);
    } else if (q.rows <= 64) {
        launchFormat<64>(ctx, p, q, g);
    } else {
        launchFormat<128>(ctx, p, q, g);
    }
}

}  // namespace b200c
