// Block-scaled 4-bit quantisation and its inverse (formats and storage: include/b200const.h).
//
// Every thread has 8 neighbours of a row: one 16-byte load of 16-bit elements, one 4-byte word of codes.
// Four threads (mxfp4) or two (nvfp4) share a block and find its largest magnitude with shuffles.
//
// One pass over the data, bound by DRAM where the values are written, too: 11008 x 4096 f16 to mxfp4 with values
// 33.6 us (6.1 TB/s of what the pass cannot do without), back to f16 19.0 us (6.0 TB/s).  Without the values it is instruction
// issue: 23.2 us (4.9 TB/s, 18.0 million instructions in 71 % of the slots), and 32.6 us for nvfp4 (28.3 million in 74 %), whose
// quotients take three instructions an element and whose blocks are half as long.
#include "mx.h"
#include "runtime.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

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
    int scaleFrom;  // nvfp4: where t comes from
    void* values;  // or nullptr
    long long valuesLd;
    long long blocks;       // blocks of a row
    long long scaleRows;    // rows of scale bytes, those that fill up the last tile included
    long long scaleBlocks;  // the same for blocks
};

enum : int {
    kScaleGiven,
    kScaleFound,    // tensorScale[1] holds the largest magnitude
    kScaleHere,     // the kernel looks for it first
    kScaleGuessed,  // tensorScale[0] is that of some of the rows; the kernel finds tensorScale[1] on its way
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

// eight 32-bit values -> eight codes, the first in the lowest nibble: nearest even, at most 6
__device__ __forceinline__ unsigned int codesOf(const float v[8]) {
    unsigned int r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// eight codes -> their values in f16 (exact), two to a word
__device__ __forceinline__ void valuesOf(unsigned int word, __half2 h[4]) {
    unsigned int r[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2*>(&r[i]);
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

// 8 elements as they lie in memory
template <class T>
struct Raw {
    static constexpr int n = 8 * sizeof(T) / 16;
    uint4 v[n];
};
// A line of 16 bytes; KEEP: it will be read again, and should stay in L2.  Volatile, and not a read-only load: what is
// read here may have been written while this kernel's CTAs waited in afterLast(), and no load may move before that.
template <bool KEEP>
__device__ __forceinline__ uint4 loadLine(const uint4* p) {
    uint4 v;
    if (KEEP) {
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    } else {
        asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    }
    return v;
}
__device__ __forceinline__ unsigned int loadWord(const unsigned char* p) {
    unsigned int v;
    asm volatile("ld.global.cs.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
// 16-byte loads that are aligned: all eight are there, or none
template <class T, bool KEEP>
__device__ __forceinline__ Raw<T> load8(const T* p, int left) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < Raw<T>::n; ++i) r.v[i] = left > 0 ? loadLine<KEEP>(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
    return r;
}

// Rows that start anywhere (aligned to their elements): memory is read and written in whole 16-byte lines all the same.
// A thread's eight elements begin m bytes into a line, m the same along a row; what it lacks of its last line is the
// first line of the next thread, and the bytes are shifted into place.  The first and last line that a warp has of
// a row hold bytes of others, too: they are read, never written whole -- a line that holds one byte of a matrix lies in
// the same allocation as that byte.
//
// N words, `bytes` (0 .. 15) on from the start of z.  A branch, since a warp's threads mostly have one row's `bytes`:
// picking the words one by one costs more than the rest.
template <int N>
__device__ __forceinline__ void shifted(const unsigned int z[N + 4], unsigned int bytes, unsigned int out[N]) {
    const unsigned int bits = (bytes & 3) * 8;
    switch (bytes >> 2) {
    case 0:
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(z[i], z[i + 1], bits);
        break;
    case 1:
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(z[i + 1], z[i + 2], bits);
        break;
    case 2:
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(z[i + 2], z[i + 3], bits);
        break;
    default:
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(z[i + 3], z[i + 4], bits);
        break;
    }
}
// hasNext: the next thread of the warp has the next eight elements of the row.  Whole warps call this.
template <class T, bool KEEP>
__device__ __forceinline__ Raw<T> loadAny(const T* p, int left, bool hasNext) {
    constexpr int n = Raw<T>::n;
    const unsigned int m = static_cast<unsigned int>(reinterpret_cast<uintptr_t>(p) & 15);
    const uint4* line = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - m);
    const int valid = min(max(left, 0), 8) * static_cast<int>(sizeof(T));
    uint4 l[n];
    if (left >= 8) {
#pragma unroll
        for (int k = 0; k < n; ++k) l[k] = loadLine<KEEP>(line + k);
    } else {
#pragma unroll
        for (int k = 0; k < n; ++k) l[k] = valid > 0 && static_cast<int>(m) + valid > 16 * k ? loadLine<KEEP>(line + k) : make_uint4(0, 0, 0, 0);
    }
    unsigned int w[4 * n + 4];
#pragma unroll
    for (int k = 0; k < n; ++k) w[4 * k] = l[k].x, w[4 * k + 1] = l[k].y, w[4 * k + 2] = l[k].z, w[4 * k + 3] = l[k].w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[4 * n + i] = __shfl_down_sync(0xFFFFFFFFu, w[i], 1);
    if ((!hasNext || left <= 8) && static_cast<int>(m) + valid > 16 * n) {
        const uint4 next = loadLine<KEEP>(line + n);
        w[4 * n] = next.x, w[4 * n + 1] = next.y, w[4 * n + 2] = next.z, w[4 * n + 3] = next.w;
    }
    Raw<T> r;
    shifted<4 * n>(w, m, reinterpret_cast<unsigned int*>(r.v));
    if (left < 8) {
        T* t = reinterpret_cast<T*>(r.v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= left) t[i] = fromFloat<T>(0.f);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void storeAny(T* p, int left, const T t[8], bool hasPrev, bool hasNext) {
    constexpr int n = Raw<T>::n, es = sizeof(T);
    const int m = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    const int valid = min(max(left, 0), 8) * es;
    const unsigned int* v = reinterpret_cast<const unsigned int*>(t);
    unsigned int z[4 * n + 4], o[4 * n];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __shfl_up_sync(0xFFFFFFFFu, v[4 * n - 4 + i], 1);
#pragma unroll
    for (int i = 0; i < 4 * n; ++i) z[4 + i] = v[i];
    shifted<4 * n>(z, (16 - m) & 15, o);
    uint4* line = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) - m);
    if (m == 0) {
#pragma unroll
        for (int i = 0; i < 4 * n; ++i) o[i] = v[i];
    }
    // the bytes of this thread's that lines take: from the start, or the second line if the first one has others' bytes
    const int from = m == 0 || hasPrev ? 0 : 16 - m;
    int to = from;
    if (left >= 8 && from == 0) {
#pragma unroll
        for (int k = 0; k < n; ++k) __stcs(line + k, make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
        to = 16 * n - m;
    } else {
#pragma unroll
        for (int k = 0; k < n; ++k) {
            if (valid >= 16 * (k + 1) - m && (k > 0 || from == 0)) {
                __stcs(line + k, make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
                to = 16 * (k + 1) - m;
            }
        }
    }
    // the next thread's first line takes the last m bytes, if it is written whole
    const int end = hasNext && (left - 8) * es >= 16 - m ? min(valid, 16 * n - m) : valid;
    if (from > 0 || to < end) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((i * es < from || i * es >= to) && i * es < end) p[i] = t[i];
    }
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw<T>& r, float v[8]) {
    const T* t = reinterpret_cast<const T*>(r.v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = toFloat<T>(t[i]);
}
// what eight codes with the factor d stand for; `POWER`: d is a power of two
template <class T, bool POWER>
__device__ __forceinline__ void values8(unsigned int word, float d, T t[8]) {
    __half2 h[4];
    valuesOf(word, h);
    if (sizeof(T) == 2 && POWER && std::is_same<T, __half>::value && d >= 5.9604645e-8f && d <= 32768.f) {
        // a factor that f16 has: the product is rounded once, and only where it is subnormal or too large
        const __half2 f = __half2half2(__float2half_rn(d));
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<__half2*>(t)[i] = __hmul2(h[i], f);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 c = __half22float2(h[i]);
            t[2 * i] = fromFloat<T>(c.x * d);
            t[2 * i + 1] = fromFloat<T>(c.y * d);
        }
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const T t[8]) {
#pragma unroll
    for (int i = 0; i < Raw<T>::n; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<const uint4*>(t)[i]);
}
// largest magnitude of the eight, as the bits of a 32-bit float: bits of magnitudes order like the magnitudes,
// for 16-bit types two at a time
template <class T>
__device__ __forceinline__ unsigned int top8(const Raw<T>& r) {
    const unsigned int* w = reinterpret_cast<const unsigned int*>(r.v);
    if (sizeof(T) == 2) {
        unsigned int m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        const unsigned short h = static_cast<unsigned short>(max(m >> 16, m & 0xFFFFu));
        return __float_as_uint(toFloat<T>(*reinterpret_cast<const T*>(&h)));
    }
    unsigned int m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
    return m;
}

// the smallest power of two t >= 2^-126 with top <= 2688 t; 2688 = 1.3125 * 2^11, so t = 2^(e - 11) when top's
// significand is at most 1.3125 and twice that otherwise
__device__ __forceinline__ float tensorScaleOf(float top) {
    if (!(top > 0.f)) return 1.f;
    const unsigned int bits = __float_as_uint(top);
    int e = static_cast<int>(bits >> 23) - 11 + ((bits & 0x7FFFFFu) > 0x280000u ? 1 : 0);
    return __uint_as_float(static_cast<unsigned int>(max(e, 1)) << 23);
}

// See mx_matmul.cu: no kernel here touches memory before the one that was launched before it has ended.
__device__ __forceinline__ void afterLast() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// How a kernel's threads lie over rows x units (8 elements): x along a row, y over rows, each thread with UNITS
// units of one row, x apart, whose loads are all under way before the first is used.  X: x where it is known, 0:
// blockDim.x.  With X = 128 the addresses of a thread's units differ by constants: with its units in different
// rows instead, 64-bit address arithmetic was a quarter of all instructions.
template <int UNITS, int X>
struct Lay {
    __device__ __forceinline__ static int x() {
        return X ? X : static_cast<int>(blockDim.x);
    }
    __device__ __forceinline__ static int firstUnit() {
        return static_cast<int>(blockIdx.y) * x() * UNITS + static_cast<int>(threadIdx.x);
    }
    __device__ __forceinline__ static int unitStep() {  // on to the next part of a row longer than the grid
        return static_cast<int>(gridDim.y) * x() * UNITS;
    }
};

// the largest finite magnitude among eight elements and `top`
template <class T>
__device__ __forceinline__ unsigned int topFinite(unsigned int top, const Raw<T>& raw) {
    const unsigned int m = top8<T>(raw);
    if (m < 0x7F800000u) return max(top, m);
    float v[8];  // a NaN or an infinity hides the others
    unpack8<T>(raw, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned int a = __float_as_uint(v[j]) & 0x7FFFFFFFu;
        if (a < 0x7F800000u) top = max(top, a);
    }
    return top;
}

// the row of the first thread of this thread's warp within its CTA
__device__ __forceinline__ int warpRow(int x) {
    const int thread = threadIdx.y * blockDim.x + threadIdx.x;
    return (thread & ~31) / x;
}

// the largest finite magnitude of this CTA's share: a warp's first thread has its result
template <class T, bool WIDE, int UNITS, int X>
__device__ __forceinline__ unsigned int topOf(const MxQuantParams& p, int lane) {
    typedef Lay<UNITS, X> L;
    constexpr int rows = UNITS > 1 ? 1 : 4;  // of a thread, whose loads are under way together
    const int x = L::x();
    const bool hasNext = (lane & (min(x, 32) - 1)) != min(x, 32) - 1;
    const int cols = static_cast<int>(p.cols), units = (cols + 7) / 8;
    const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
    unsigned int top = 0;
    // rows of the warp's first thread
    for (long long r0 = static_cast<long long>(blockIdx.x) * blockDim.y + warpRow(x); r0 < p.rows; r0 += rows * step) {
        for (int base = L::firstUnit() - static_cast<int>(threadIdx.x); base < units; base += L::unitStep()) {
            const int u = base + threadIdx.x;
            Raw<T> raw[UNITS * rows];
#pragma unroll
            for (int i = 0; i < UNITS * rows; ++i) {
                const int ui = u + (UNITS > 1 ? i * x : 0);
                const long long r = r0 + (UNITS > 1 ? 0 : i * step) + (x < 32 ? lane / x : 0);
                const T* from = static_cast<const T*>(p.src) + r * p.srcLd + ui * 8ll;
                const int left = r < p.rows ? cols - 8 * ui : 0;
                raw[i] = WIDE ? load8<T, true>(from, left) : loadAny<T, true>(from, left, hasNext);
            }
#pragma unroll
            for (int i = 0; i < UNITS * rows; ++i) top = topFinite<T>(top, raw[i]);
        }
    }
    return __reduce_max_sync(0xFFFFFFFFu, top);
}

// A memset in the stream would end the kernels' overlapping: 3 us more.
__global__ void mxZeroKernel(float* tensorScale) {
    afterLast();
    if (threadIdx.x < 2) tensorScale[threadIdx.x] = 0.f;
}

// -> tensorScale[1], zeroed before.  A maximum does not depend on the order it is taken in.
template <class T, bool WIDE, int UNITS, int X>
__global__ void __launch_bounds__(256) mxTopKernel(const __grid_constant__ MxQuantParams p) {
    __shared__ unsigned int tops[8];
    afterLast();
    const int thread = threadIdx.y * Lay<UNITS, X>::x() + threadIdx.x, lane = thread & 31, warps = blockDim.x * blockDim.y / 32;
    unsigned int top = topOf<T, WIDE, UNITS, X>(p, lane);
    if (lane == 0) tops[thread >> 5] = top;
    __syncthreads();
    if (thread < 32) {
        top = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? tops[lane] : 0u);
        if (lane == 0 && top) atomicMax(reinterpret_cast<unsigned int*>(p.tensorScale) + 1, top);
    }
}

// One cluster of CTAs: its first one collects the others' results, and nothing has to be zeroed before.
template <class T, bool WIDE, int UNITS, int X>
__global__ void __launch_bounds__(256) mxTopClusterKernel(const __grid_constant__ MxQuantParams p) {
    __shared__ unsigned int tops[8];
    afterLast();
    const int thread = threadIdx.y * Lay<UNITS, X>::x() + threadIdx.x, lane = thread & 31, warps = blockDim.x * blockDim.y / 32;
    const unsigned int top = topOf<T, WIDE, UNITS, X>(p, lane);
    if (lane == 0) tops[thread >> 5] = top;
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (blockIdx.x == 0 && thread < 32) {
        unsigned int all = 0;
        for (int i = lane; i < warps * static_cast<int>(gridDim.x); i += 32) {
            unsigned int at, v;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<unsigned int>(__cvta_generic_to_shared(tops + i % warps))), "r"(i / warps));
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
            all = max(all, v);
        }
        all = __reduce_max_sync(0xFFFFFFFFu, all);
        if (lane == 0) {
            // for a guess; of zeros the smallest that there is: that of the whole matrix may be any
            p.tensorScale[0] = all ? tensorScaleOf(__uint_as_float(all)) : 1.17549435e-38f;
            p.tensorScale[1] = __uint_as_float(all);
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The same by one CTA alone, for a small matrix: this thread's warp's share.
template <class T, bool WIDE>
__device__ __forceinline__ unsigned int topHere(const MxQuantParams& p, int thread, int threads) {
    constexpr int batch = WIDE ? 4 : 2, each = WIDE ? 8 : 1;  // of 8 elements under way at once; neighbours of one load
    const int cols = static_cast<int>(p.cols), across = (cols + each - 1) / each, n = static_cast<int>(p.rows) * across;
    unsigned int top = 0;
    for (int first = thread; first < n; first += threads * batch * 8 / each) {
        Raw<T> raw[batch];
#pragma unroll
        for (int i = 0; i < batch * 8 / each; ++i) {
            const int at = first + i * threads, r = at / across, c = at - r * across;
            const T* from = static_cast<const T*>(p.src) + r * p.srcLd + c * each;
            if (WIDE) {
                raw[i] = load8<T, true>(from, at < n ? 8 : 0);
            } else {
                reinterpret_cast<T*>(raw)[i] = at < n ? *from : fromFloat<T>(0.f);
            }
        }
#pragma unroll
        for (int i = 0; i < batch; ++i) top = topFinite<T>(top, raw[i]);
    }
    return __reduce_max_sync(0xFFFFFFFFu, top);
}

// v / d in 32 bits, as codes and scales need it.  The method is Markstein's (Computation of elementary functions on the IBM
// RISC System/6000 processor, IBM Journal of Research and Development 34, 1990): a reciprocal r by one Newton-Raphson
// step, and the quotient q = v r corrected once by its remainder, q + (v - q d) r.  With the
// division of the language instead 11008 x 4096 f16 to nvfp4, codes only, takes 45.5 us, not 32.6.
// With r off by 2^-23 at most (the approximation's error squared, and one rounding) q is off by 1.5 * 2^-23, and the sum
// before its last rounding by the product of the two: less than 2^-44 of v / d.  That is less than correct rounding, but
// enough for what is read from it, the side of a border between two codes or scales (or the border itself) that the rounded
// quotient lies on.  A border b has up to five significant bits.  With d brought to 1 .. 2 and v along, v - d b is a
// multiple of 2^-27, and the two roundings differ only if v is within 2^-42 of d times the middle between b and the next
// number, 2^-24 away: only if d lies within 2^-18 of a multiple of 1/8.  Of these few divisors the tests try each with
// every border's neighbours, and find none whose code or scale is not that of the correctly rounded quotient.  For d of
// four bits, that is for t a power of two as the one found here, nothing has to be tried: v is d b, or differs from it by
// a unit in its last place, and v / d stays 0.03 units away from the middle.
// The remainder is exact enough for d and v within 2^-60 .. 2^60; quotients below 2^-20, for which it may not be, are the
// code and the scale 0 either way.  Otherwise d is brought to 1 .. 2 first and v along with it; what then leaves 32 bits
// is far above the largest code or below the smallest.
struct Divisor {
    float d, r, s1, s2;
    bool far;
    __device__ __forceinline__ Divisor(float by, float top): d(by), s1(1.f), s2(1.f) {
        far = !(by >= 8.6736174e-19f && by <= 1.1529215e18f && top <= 1.1529215e18f);
        if (far) {
            if (by <= 3.402823466e38f) {
                const float n = by < 1.1754944e-38f ? by * 16777216.f : by;  // subnormal numbers have no exponent field
                const int e = static_cast<int>(__float_as_uint(n) >> 23) - 127 - (by < 1.1754944e-38f ? 24 : 0);
                const int h = -e / 2;
                s1 = __uint_as_float(static_cast<unsigned int>(h + 127) << 23);
                s2 = __uint_as_float(static_cast<unsigned int>(-e - h + 127) << 23);
                d = by * s1 * s2;
            } else {  // infinity: all quotients are 0
                s1 = 0.f;
                d = 1.f;
            }
        }
        float r0;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d));
        r = __fmaf_rn(__fmaf_rn(-d, r0, 1.f), r0, r0);
    }
    __device__ __forceinline__ float near(float v) const {
        // the remainder is taken with its sign turned: the other way round -0 would become 0
        const float q = __fmul_rn(v, r);
        return __fmaf_rn(-__fmaf_rn(q, d, -v), r, q);
    }
    __device__ __forceinline__ float within(float v) const {
        return fminf(fmaxf(v * s1 * s2, -1e30f), 1e30f);
    }
};

// Eight elements of a block whose largest magnitude is `top` -> their codes; the block's scale and the factor of
// its codes (which makes NaN of the codes of a block with a NaN or an infinity).
template <class T, bool NV>
__device__ __forceinline__ unsigned int encode8(const Raw<T>& raw, unsigned int top, float t, const Divisor& sixT, bool badT, unsigned int* scaleByte,
                                                float* factor) {
    const bool poison = top >= 0x7F800000u;
    float v[8];
    unpack8<T>(raw, v);
    bool zero = poison;
    if (!NV) {
        // the exponent field of the largest magnitude, less 2; subnormal numbers have the field 0
        const unsigned int scale = poison ? 0xFFu : static_cast<unsigned int>(max(static_cast<int>(top >> 23) - 2, 0));
        const float up = __uint_as_float((254u << 23) - (scale << 23));  // 2^-X
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * up;
        *scaleByte = scale;
        // 2^X, a subnormal number for the byte 0; infinity for 0xFF, and the codes are 0
        *factor = __uint_as_float(max(scale << 23, 0x00400000u));
    } else {
        const float m = __uint_as_float(top);
        const float s = sixT.near(sixT.far || !(m <= 1.1529215e18f) ? sixT.within(m) : m);
        const unsigned int scale = poison || badT ? 0x7Fu : toE4m3(fminf(s, 448.f));
        const float d = __fmul_rn(fromE4m3(scale), t);
        zero = scale == 0x7Fu || !(d > 0.f);
        const Divisor by(d, m);
        if (by.far) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = by.within(v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = by.near(v[i]);
        *scaleByte = scale;
        *factor = d;
    }
    const unsigned int word = codesOf(v);
    return zero ? 0u : word;
}

// Whole warps go through the loop together, whatever their rows.  The last CTAs of the grid (blockIdx.x >=
// rowCtas) zero the scales of the rows that only fill a tile up.
template <class T, bool NV, bool WIDE, bool VALUES, int UNITS, int X>
__global__ void __launch_bounds__(256, 4) mxQuantKernel(const __grid_constant__ MxQuantParams p, int rowCtas) {
    typedef Lay<UNITS, X> L;
    __shared__ unsigned int tops[8];
    afterLast();
    const int x = L::x(), thread = threadIdx.y * x + threadIdx.x, lane = thread & 31, warp = thread >> 5;
    if (static_cast<int>(blockIdx.x) >= rowCtas) {
        const int threads = blockDim.x * blockDim.y;
        const long long chunks = p.scaleBlocks / 4, n = (p.scaleRows - p.rows) * chunks;
        const long long cta = static_cast<long long>(blockIdx.x - rowCtas) * gridDim.y + blockIdx.y;
        const long long all = static_cast<long long>(gridDim.x - rowCtas) * gridDim.y * threads;
        for (long long i = cta * threads + thread; i < n; i += all) {
            *reinterpret_cast<unsigned int*>(p.scales + scaleAt(1, p.rows + i / chunks, i % chunks * 4, p.blocks)) = 0u;
        }
        return;
    }
    float t = 1.f;
    if (NV) {
        if (p.scaleFrom == kScaleGiven || p.scaleFrom == kScaleGuessed) {
            t = p.tensorScale[0];
        } else {
            float top;
            if (p.scaleFrom == kScaleHere) {
                const unsigned int mine = topHere<T, WIDE>(p, thread, blockDim.x * blockDim.y);
                if (lane == 0) tops[warp] = mine;
                __syncthreads();
                unsigned int all = 0;
                for (int i = 0; i < static_cast<int>(blockDim.x * blockDim.y) / 32; ++i) all = max(all, tops[i]);
                top = __uint_as_float(all);
            } else {
                top = p.tensorScale[1];
            }
            t = tensorScaleOf(top);
            if (blockIdx.x == 0 && blockIdx.y == 0 && thread == 0) {
                p.tensorScale[0] = t;
                if (p.scaleFrom == kScaleHere) p.tensorScale[1] = top;
            }
        }
    }
    const Divisor sixT(NV ? 6.f * t : 1.f, 0.f);
    const bool badT = NV && !(t > 0.f && t <= 3.402823466e38f);
    constexpr int lanes = NV ? 2 : 4;  // threads of a block
    const int cols = static_cast<int>(p.cols), units = (cols + 31) / 32 * 4;
    const int all = max(units, static_cast<int>(p.scaleBlocks) * lanes);  // those of a tile's filling scales too
    // from the last row to the first: where the largest magnitude was looked for just before, the last rows are
    // what L2 still holds (11008 x 4096 f16: 65.6 -> 62.5 us for both kernels)
    const long long r = p.rows - 1 - (static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y);
    const int run = min(x, 32);  // threads of a warp that lie in one row
    const bool hasPrev = (lane & (run - 1)) != 0, hasNext = (lane & (run - 1)) != run - 1;
    const T* src = static_cast<const T*>(p.src) + r * p.srcLd;
    unsigned char* codes = p.codes + r * p.ld;
    T* values = static_cast<T*>(p.values) + r * p.valuesLd;
    // tiled: blocks of four lie 512 bytes apart
    unsigned char* scales = p.scales + (r >= 0 ? scaleAt(p.tiled, r, 0, p.blocks) : 0);
    const bool watch = NV && p.scaleFrom == kScaleGuessed;
    unsigned int seen = 0;  // the largest finite magnitude
    const int begin = L::firstUnit() - static_cast<int>(threadIdx.x);
    for (int base = begin; base < all; base += L::unitStep()) {
        const int u = base + threadIdx.x;
        Raw<T> raw[UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const T* from = src + u * 8ll + i * x * 8;
            const int left = r >= 0 ? cols - 8 * (u + i * x) : 0;
            raw[i] = WIDE ? load8<T, false>(from, left) : loadAny<T, false>(from, left, hasNext);
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int ui = u + i * x, left = cols - 8 * ui;
            unsigned int top = top8<T>(raw[i]);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            if (!NV) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            if (watch) seen = top < 0x7F800000u ? max(seen, top) : topFinite<T>(seen, raw[i]);
            float d;
            unsigned int scale;
            const unsigned int word = encode8<T, NV>(raw[i], top, t, sixT, badT, &scale, &d);
            if (r >= 0) {
                const int b = ui / lanes;
                if ((ui & (lanes - 1)) == 0 && b < p.scaleBlocks) {
                    scales[p.tiled ? (b >> 2) * 512ll + (b & 3) : b] = static_cast<unsigned char>(left > 0 ? scale : 0u);
                }
                if (ui < units) *reinterpret_cast<unsigned int*>(codes + ui * 4ll) = word;
            }
            if (VALUES) {
                alignas(16) T w[8];
                values8<T, !NV>(word, d, w);
                if (WIDE) {
                    if (r >= 0 && left > 0) store8<T>(values + ui * 8ll, w);
                } else {
                    storeAny<T>(values + ui * 8ll, r >= 0 ? left : 0, w, hasPrev, hasNext);
                }
            }
        }
    }
    if (watch) {
        seen = __reduce_max_sync(0xFFFFFFFFu, seen);
        if (lane == 0) tops[warp] = seen;
        __syncthreads();
        if (thread == 0) {
            for (int i = 1; i < static_cast<int>(blockDim.x * blockDim.y) / 32; ++i) seen = max(seen, tops[i]);
            unsigned int* word = reinterpret_cast<unsigned int*>(p.tensorScale) + 1;
            if (seen > *reinterpret_cast<volatile unsigned int*>(word)) atomicMax(word, seen);  // few are
        }
    }
}

// After a guessed factor: where the one that the whole matrix gives is 2^k times it, a block's scale is 2^-k times
// what was stored, with the same codes and values, as long as neither is at the ends of what e4m3 holds: between them
// its rounding is relative to the number.  The guess is that of some of the rows, so k > 0; a scale of 0 then stays 0
// and NaN stays NaN.  The blocks at the ends, mostly few, are quantised again.  Scales are walked in the order that
// they are stored in: row by row, tiled ones took 122 us (32000 x 4096) for sectors of which a warp used four bytes.
template <class T>
__global__ void __launch_bounds__(256) mxRepairKernel(const __grid_constant__ MxQuantParams p) {
    afterLast();
    const float guess = p.tensorScale[0], t = tensorScaleOf(p.tensorScale[1]);
    if (t == guess) return;
    const int k = static_cast<int>(__float_as_uint(t) >> 23) - static_cast<int>(__float_as_uint(guess) >> 23);
    const Divisor sixT(6.f * t, 0.f);
    const int lane = threadIdx.x & 31;
    const long long n = p.scaleRows * p.scaleBlocks;
    const int each = reinterpret_cast<uintptr_t>(p.scales) % 16 == 0 ? 16 : 1;  // scales of a thread
    const long long step = static_cast<long long>(gridDim.x) * blockDim.x * each;
    // whole warps go through the loop together
    for (long long at = (static_cast<long long>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31)) * each; at < n; at += step) {
        const long long mine = at + lane * each;
        const int count = static_cast<int>(max(0ll, min(static_cast<long long>(each), n - mine)));
        alignas(16) unsigned char s[16];
        if (count == 16) {
            *reinterpret_cast<uint4*>(s) = *reinterpret_cast<const uint4*>(p.scales + mine);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = j < count ? p.scales[mine + j] : 0;
        }
        unsigned int again = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int b = s[j], moved = b - 8 * k;
            if (b != 0 && b != 0x7F) {
                if (b < 8 || b > 125 || moved < 8) {
                    again |= 1u << j;
                } else {
                    s[j] = static_cast<unsigned char>(moved);
                }
            }
        }
        if (count == 16) {
            *reinterpret_cast<uint4*>(p.scales + mine) = *reinterpret_cast<const uint4*>(s);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < count) p.scales[mine + j] = s[j];
        }
        __syncwarp();
        // one thread's blocks after another's, two threads to each
        for (unsigned int todo = __ballot_sync(0xFFFFFFFFu, again != 0); todo; todo &= todo - 1) {
            const int from = __ffs(todo) - 1;
            const bool on = __shfl_sync(0xFFFFFFFFu, again, from) >> (lane / 2) & 1;
            const long long i = at + from * each + lane / 2;
            long long row, b;
            if (p.tiled) {
                const long long tile = i / 512, chunks = p.scaleBlocks / 4;
                const int in = static_cast<int>(i % 512);
                row = tile / chunks * 128 + in % 16 / 4 * 32 + in / 16;
                b = tile % chunks * 4 + in % 4;
            } else {
                row = i / p.blocks;
                b = i % p.blocks;
            }
            const long long u = b * 2 + (lane & 1);  // eight elements
            const int left = on ? static_cast<int>(min(8ll, p.cols - 8 * u)) : 0;
            Raw<T> raw;
            T* e = reinterpret_cast<T*>(raw.v);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = j < left ? static_cast<const T*>(p.src)[row * p.srcLd + u * 8 + j] : fromFloat<T>(0.f);
            unsigned int top = top8<T>(raw);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            float d;
            unsigned int scale;
            const unsigned int word = encode8<T, true>(raw, top, t, sixT, false, &scale, &d);
            if (left > 0) {
                if ((lane & 1) == 0) p.scales[i] = static_cast<unsigned char>(scale);
                *reinterpret_cast<unsigned int*>(p.codes + row * p.ld + u * 4) = word;
                if (p.values) {
                    alignas(16) T w[8];
                    values8<T, false>(word, d, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) static_cast<T*>(p.values)[row * p.valuesLd + u * 8 + j] = w[j];
                }
            }
        }
    }
}
__global__ void mxScaleKernel(float* tensorScale) {
    afterLast();
    if (threadIdx.x == 0) tensorScale[0] = tensorScaleOf(tensorScale[1]);
}

template <class T, bool NV, bool WIDE, int UNITS, int X>
__global__ void __launch_bounds__(256) mxDequantKernel(const __grid_constant__ MxDequantParams p) {
    typedef Lay<UNITS, X> L;
    afterLast();
    const int x = L::x(), lane = (threadIdx.y * x + threadIdx.x) & 31;
    const int run = min(x, 32);
    const bool hasPrev = (lane & (run - 1)) != 0, hasNext = (lane & (run - 1)) != run - 1;
    const float t = NV ? p.tensorScale[0] : 1.f;
    const int cols = static_cast<int>(p.cols), units = (cols + 7) / 8;
    const long long r = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool row = r < p.rows;
    const unsigned char* codes = p.codes + r * p.ld;
    const unsigned char* scales = p.scales + (row ? scaleAt(p.tiled, r, 0, p.blocks) : 0);
    T* out = static_cast<T*>(p.out) + r * p.outLd;
    for (int base = L::firstUnit() - static_cast<int>(threadIdx.x); base < units; base += L::unitStep()) {
        const int u = base + threadIdx.x;
        unsigned int word[UNITS], scale[UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int ui = u + i * x;
            word[i] = scale[i] = 0;
            if (row && ui < units) {
                const int b = ui / (NV ? 2 : 4);
                word[i] = loadWord(codes + ui * 4ll);
                scale[i] = scales[p.tiled ? (b >> 2) * 512ll + (b & 3) : b];
            }
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int ui = u + i * x;
            const float d = NV ? __fmul_rn(fromE4m3(scale[i]), t) : fromE8m0(scale[i]);
            alignas(16) T w[8];
            values8<T, !NV>(word[i], d, w);
            if (WIDE) {
                if (row && ui < units) store8<T>(out + ui * 8ll, w);
            } else {
                storeAny<T>(out + ui * 8ll, row ? cols - 8 * ui : 0, w, hasPrev, hasNext);
            }
        }
    }
}

// rows x units of 8 elements over CTAs
void gridFor(long long rows, int x, int threads, long long along, long long units, dim3* grid, dim3* block) {
    *block = dim3(x, threads / x);
    *grid = dim3(static_cast<unsigned int>(std::max<long long>(1, (rows + block->y - 1) / block->y)),
                 static_cast<unsigned int>(std::max<long long>(1, std::min<long long>((units + along - 1) / along, 65535))));
}

// Which form of a kernel: threads with four units of a row where there are enough threads to fill the SMs (four CTAs
// each) all the same, 128 along a row or -- shorter rows, or rows that would leave many of 128 idle -- fewer.
struct Form {
    int units, x;
    bool fixed;  // X = 128
};
Form formFor(Context* ctx, long long rows, long long units) {
    Form f{1, 4, false};
    if (units > 8 && rows * units >= 256ll * 4 * 4 * ctx->smCount) {
        f.units = 4;
        long long idle = -1;
        for (int x = 128; x >= 4; x /= 2) {
            const long long along = 4ll * x, padded = (units + along - 1) / along * along;
            if (idle < 0 || padded * 8 < idle * 7) {  // an eighth fewer is worth the shorter stretch
                idle = padded;
                f.x = x;
            }
        }
        f.fixed = f.x == 128;
    } else {
        while (f.x < 256 && f.x < units) f.x *= 2;
    }
    return f;
}
template <class F>
void withForm(const Form& f, F&& run) {
    if (f.fixed) {
        run(std::integral_constant<int, 4>(), std::integral_constant<int, 128>());
    } else if (f.units == 4) {
        run(std::integral_constant<int, 4>(), std::integral_constant<int, 0>());
    } else {
        run(std::integral_constant<int, 1>(), std::integral_constant<int, 0>());
    }
}

template <class Kernel, class... Args>
void launchNext(Context* ctx, Kernel kernel, dim3 grid, dim3 block, int cluster, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    ++ctx->launches;
}

bool aligned16(const void* p, long long ldBytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ldBytes % 16 == 0;
}

template <class T, bool WIDE>
void findTop(Context* ctx, const MxQuantParams& p) {  // -> tensorScale[1]; of up to 1 MB [0] as well
    const long long units = (p.cols + 7) / 8;
    const Form f = formFor(ctx, p.rows, units);
    dim3 grid, block;
    gridFor(p.rows, f.x, f.fixed ? 128 : 256, static_cast<long long>(f.x) * f.units, units, &grid, &block);
    // eight CTAs read about 1 MB in the time that zeroing the word and a grid's atomics take
    const bool cluster = p.rows * units * 8 * static_cast<long long>(sizeof(T)) <= (1ll << 20);
    if (!cluster) launchNext(ctx, mxZeroKernel, dim3(1), dim3(32), 1, p.tensorScale);
    // all atomics go to one word, one after another: one for each of few CTAs (one for each warp of many took 16 us for
    // 1024 x 4096)
    grid.x = cluster ? 8u : std::min<unsigned int>(grid.x, ctx->smCount * (f.fixed ? 8u : 4u));
    if (cluster) grid.y = 1;
    withForm(f, [&](auto n, auto x) {
        if (cluster) {
            launchNext(ctx, mxTopClusterKernel<T, WIDE, decltype(n)::value, decltype(x)::value>, grid, block, 8, p);
        } else {
            launchNext(ctx, mxTopKernel<T, WIDE, decltype(n)::value, decltype(x)::value>, grid, block, 1, p);
        }
    });
}

template <class T, bool NV, bool WIDE>
void quantizeWith(Context* ctx, const MxQuantParams& p) {
    if (NV && p.scaleFrom == kScaleFound) findTop<T, WIDE>(ctx, p);
    if (NV && p.scaleFrom == kScaleGuessed) {
        MxQuantParams some = p;  // rows far from one another, less than 1 MB in all
        const long long every = (p.rows * ((p.cols + 7) / 8 * 8) * static_cast<long long>(sizeof(T)) >> 20) + 1;
        some.rows = std::max<long long>(1, p.rows / every);
        some.srcLd = p.srcLd * every;
        findTop<T, WIDE>(ctx, some);
    }
    // an empty matrix has no scales, but its factor is still written
    const long long units = std::max((p.cols + 31) / 32 * 4, p.scaleBlocks * (NV ? 2 : 4));
    if ((p.rows == 0 || units == 0) && !(NV && p.scaleFrom != kScaleGiven)) return;
    const Form f = formFor(ctx, p.rows, units);
    dim3 grid, block;
    gridFor(p.rows, f.x, f.fixed ? 128 : 256, static_cast<long long>(f.x) * f.units, units, &grid, &block);
    const int rowCtas = static_cast<int>(grid.x);
    if (p.scaleRows > p.rows) {
        const long long words = (p.scaleRows - p.rows) * (p.scaleBlocks / 4), perX = static_cast<long long>(block.x) * block.y * grid.y;
        grid.x += static_cast<unsigned int>(std::min<long long>((words + perX - 1) / perX, 1024));
    }
    withForm(f, [&](auto n, auto x) {
        if (p.values) {
            launchNext(ctx, mxQuantKernel<T, NV, WIDE, true, decltype(n)::value, decltype(x)::value>, grid, block, 1, p, rowCtas);
        } else {
            launchNext(ctx, mxQuantKernel<T, NV, WIDE, false, decltype(n)::value, decltype(x)::value>, grid, block, 1, p, rowCtas);
        }
    });
    if (NV && p.scaleFrom == kScaleGuessed) {
        launchNext(ctx, mxRepairKernel<T>, dim3(ctx->smCount * 8u), dim3(256), 1, p);
        launchNext(ctx, mxScaleKernel, dim3(1), dim3(32), 1, p.tensorScale);
    }
}

template <class T>
void quantizeAs(Context* ctx, const MxQuantParams& p, bool nv) {
    // eight columns at a time, all of them there: 16-byte accesses
    const bool wide = p.cols % 8 == 0 && aligned16(p.src, p.srcLd * sizeof(T)) && (!p.values || aligned16(p.values, p.valuesLd * sizeof(T)));
    if (nv) {
        wide ? quantizeWith<T, true, true>(ctx, p) : quantizeWith<T, true, false>(ctx, p);
    } else {
        wide ? quantizeWith<T, false, true>(ctx, p) : quantizeWith<T, false, false>(ctx, p);
    }
}

template <class T, bool NV, bool WIDE>
void dequantizeWith(Context* ctx, const MxDequantParams& p) {
    const long long units = (p.cols + 7) / 8;
    const Form f = formFor(ctx, p.rows, units);
    dim3 grid, block;
    gridFor(p.rows, f.x, f.fixed ? 128 : 256, static_cast<long long>(f.x) * f.units, units, &grid, &block);
    withForm(f, [&](auto n, auto x) {
        launchNext(ctx, mxDequantKernel<T, NV, WIDE, decltype(n)::value, decltype(x)::value>, grid, block, 1, p);
    });
}

template <class T>
void dequantizeAs(Context* ctx, const MxDequantParams& p, bool nv) {
    const bool wide = p.cols % 8 == 0 && aligned16(p.out, p.outLd * sizeof(T));
    if (nv) {
        wide ? dequantizeWith<T, true, true>(ctx, p) : dequantizeWith<T, true, false>(ctx, p);
    } else {
        wide ? dequantizeWith<T, false, true>(ctx, p) : dequantizeWith<T, false, false>(ctx, p);
    }
}

}  // namespace

void launchMxQuantize(Context* ctx, const void* src, int dtype, int64_t srcLd, const b200c_mx_matrix& out, void* values,
                      int64_t valuesLd, bool scaleGiven) {
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
    // Up to 64 KB every CTA looks the matrix through by itself: 16 loads of a thread, where two launches before this
    // one take about 5 us.  From 128 MB on, when most of the second read would not come from L2 either, the matrix is
    // read once, with a guess that is put right afterwards (f32 with values, 32000 x 4096: 275 -> 196 us, 8192 x 8192:
    // 141 -> 99; f16 of 64 MB: 40 -> 47 us, of 90 MB: 56 -> 58).  The guess looks at whole rows, so they are at most a
    // quarter of what it may read.
    const int64_t bytes = out.rows * ((out.cols + 7) / 8 * 8) * (dtBits(dtype) / 8);
    p.scaleFrom = scaleGiven                                                       ? kScaleGiven
                  : bytes <= 65536                                                 ? kScaleHere
                  : bytes >= (128ll << 20) && out.cols * (dtBits(dtype) / 8) <= (1ll << 18) ? kScaleGuessed
                                                                                   : kScaleFound;
    p.values = values;
    p.valuesLd = valuesLd;
    p.blocks = mxBlocks(out.format, out.cols);
    p.scaleRows = out.cols == 0 ? 0 : p.tiled ? roundUp(out.rows, 128) : out.rows;
    p.scaleBlocks = p.tiled ? roundUp(p.blocks, 4) : p.blocks;
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
