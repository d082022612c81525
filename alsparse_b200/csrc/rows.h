// What the operators on rows of dense blocks (embedding.cu, route.cu, experts.cu, expert_mm.cu) share: element types,
// vector access, checks of arguments.  Not part of the C ABI.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"

namespace asb {

// ---- element types ---------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

template <typename T> __device__ __forceinline__ unsigned pack_two(float a, float b);  // 16-bit types, a in the low half
template <> __device__ __forceinline__ unsigned pack_two<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&v);
}
template <> __device__ __forceinline__ unsigned pack_two<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&v);
}

// N consecutive elements as words, moved in accesses of at most 16 bytes.  (Kept as words and taken apart by shifts: arrays of
// 16-bit elements cost the compiler registers and stack.)
template <typename T, int N>
struct Pack {
    static constexpr int bytes = sizeof(T) * N, words = bytes < 4 ? 1 : bytes / 4;
    unsigned w[words];
};

// PLAIN: memory that the kernel writes too
template <typename T, int N, bool PLAIN = false>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    Pack<T, N> r;
    constexpr int bytes = Pack<T, N>::bytes;
    const auto get = [](const auto *q) { return PLAIN ? *q : __ldg(q); };
    if constexpr (bytes >= 16) {
#pragma unroll
        for (int i = 0; i < bytes / 16; i++) {
            const uint4 v = get(reinterpret_cast<const uint4 *>(p) + i);
            r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (bytes == 8) {
        const uint2 v = get(reinterpret_cast<const uint2 *>(p));
        r.w[0] = v.x, r.w[1] = v.y;
    } else if constexpr (bytes == 4) {
        r.w[0] = get(reinterpret_cast<const unsigned *>(p));
    } else {
        r.w[0] = get(reinterpret_cast<const unsigned short *>(p));
    }
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r) {
    constexpr int bytes = Pack<T, N>::bytes;
    if constexpr (bytes >= 16) {
#pragma unroll
        for (int i = 0; i < bytes / 16; i++)
            reinterpret_cast<uint4 *>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
    } else if constexpr (bytes == 8) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
    } else if constexpr (bytes == 4) {
        *reinterpret_cast<unsigned *>(p) = r.w[0];
    } else {
        *reinterpret_cast<unsigned short *>(p) = (unsigned short)r.w[0];
    }
}

// All bits zero: zeros of every type
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> zero_pack() {
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < Pack<T, N>::words; i++) r.w[i] = 0;
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N> &p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (std::is_same<T, float>::value) {
            f[i] = __uint_as_float(p.w[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            f[i] = __uint_as_float(i & 1 ? p.w[i / 2] & 0xffff0000u : p.w[i / 2] << 16);
        } else {
            f[i] = __half2float(__ushort_as_half((unsigned short)(i & 1 ? p.w[i / 2] >> 16 : p.w[i / 2] & 0xffffu)));
        }
    }
}

// Rounds to nearest, ties to even: the only rounding to the type
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&f)[N]) {
    Pack<T, N> r;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < N; i++) r.w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < (N + 1) / 2; i++) r.w[i] = pack_two<T>(f[2 * i], 2 * i + 1 < N ? f[2 * i + 1] : 0.f);
    }
    return r;
}

// ---- rows that begin on no 16-byte boundary ------------------------------------------------------

// The memory of an operand: aligned loads around one of its rows do not reach out of it.
struct Window {
    const char *lo, *hi;
};

// The 16 bytes that begin `shift` bytes into two aligned vectors
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> across(const uint4 &x, const uint4 &y, unsigned shift) {
    Pack<T, 16 / sizeof(T)> r;
    unsigned c[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 6; i++) c[i] = shift & 8 ? c[i + 2] : c[i];
#pragma unroll
    for (int i = 0; i < 5; i++) c[i] = shift & 4 ? c[i + 1] : c[i];
#pragma unroll
    for (int i = 0; i < 4; i++) r.w[i] = sizeof(T) == 4 ? c[i] : __funnelshift_r(c[i], c[i + 1], (shift & 2) * 8);
    return r;
}

template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> one_by_one(const T *p, int n) {
    constexpr int E = 16 / sizeof(T);
    Pack<T, E> r = zero_pack<T, E>();
#pragma unroll
    for (int i = 0; i < E; i++)
        if (i < n) {
            if constexpr (sizeof(T) == 4) r.w[i] = __ldg(reinterpret_cast<const unsigned *>(p) + i);
            else r.w[i / 2] |= (unsigned)__ldg(reinterpret_cast<const unsigned short *>(p) + i) << (i & 1) * 16;
        }
    return r;
}

// n elements, 16 bytes at most, from an address that is only aligned to the element: the two aligned vectors that hold them,
// shifted together; element by element where those reach out of the operand.  What comes behind the n is nobody's.
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> load_any(const T *p, int n, const Window &w) {
    constexpr int E = 16 / sizeof(T);
    const unsigned shift = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15);
    const char *a = reinterpret_cast<const char *>(p) - shift;
    if (shift == 0 && n == E) return load_pack<T, E>(p);
    if (a < w.lo || a + 32 > w.hi) return one_by_one<T>(p, n);
    return across<T>(__ldg(reinterpret_cast<const uint4 *>(a)), __ldg(reinterpret_cast<const uint4 *>(a) + 1), shift);
}

__device__ __forceinline__ uint4 load_if(const void *p, bool there) {
    uint4 v = make_uint4(0, 0, 0, 0);
    asm("{\n.reg .pred p;\nsetp.ne.b32 p, %5, 0;\n@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
        : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
        : "l"(p), "r"((unsigned)there));
    return v;
}

// 16 bytes as load_any gives them, in two parts: the two aligned vectors are requested without a branch, so that several are on
// their way at once, and shifted together when they are needed.  `there` false: zeros.  (Experts' products of 32,768 x 1001 x 1439,
// 16 experts: 1346 us with load_any and eight warps, 876 us so, about 870 with fourteen.  The kernels on rows, which have more
// blocks to hide latency, lose by the registers: combine of rows of 2047 94 -> 127 us.)
template <typename T>
struct AnyPack {
    static constexpr int E = 16 / sizeof(T);
    uint4 x, y;
    const T *p;
    bool apart;
    __device__ __forceinline__ AnyPack() {}
    __device__ __forceinline__ AnyPack(const T *p_, const Window &w, bool there) : p(p_) {
        const unsigned shift = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15);
        const char *a = reinterpret_cast<const char *>(p) - shift;
        const bool inside = shift == 0 || (a >= w.lo && a + 32 <= w.hi);
        x = load_if(a, there && inside);
        y = load_if(a + 16, there && inside && shift != 0);
        apart = there && !inside;
    }
    __device__ __forceinline__ Pack<T, E> get() const {
        return apart ? one_by_one<T>(p, E) : across<T>(x, y, (unsigned)(reinterpret_cast<uintptr_t>(p) & 15));
    }
};

// The first n elements of a pack to where a row ends or begins; all of it, where n says so, to a 16-byte boundary
template <typename T>
__device__ __forceinline__ void store_any(T *p, int n, const Pack<T, 16 / sizeof(T)> &v) {
    constexpr int E = 16 / sizeof(T);
    if (n == E) {
        store_pack<T, E>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < E; i++)
        if (i < n) {
            if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned *>(p)[i] = v.w[i];
            else reinterpret_cast<unsigned short *>(p)[i] = (unsigned short)(v.w[i / 2] >> (i & 1) * 16);
        }
}

// A row of `width` elements cut at the 16-byte boundaries of memory: piece 0 up to the first, then pieces of 16 bytes, the last
// of what is left, and empty ones.
template <typename T>
struct Cut {
    static constexpr int E = 16 / sizeof(T);
    int head, width;
    __device__ __forceinline__ Cut(const T *row, int width_) : width(width_) {
        head = min(width, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
    }
    __device__ __forceinline__ int begin(int v) const { return v == 0 ? 0 : min(width, head + (v - 1) * E); }
    __device__ __forceinline__ int count(int v) const { return v == 0 ? head : min(width, head + v * E) - begin(v); }
};
// Pieces of a row, whichever way it is cut
inline int64_t most_pieces(int64_t width, size_t elem) { return width * (int64_t)elem / 16 + 2; }

// ---- launches ----------------------------------------------------------------------------------

// A kernel that begins with after_previous(): its blocks may be made resident while the kernel before it on the stream ends
// (as soon as that one has called let_next_begin or its blocks are done), and wait there until its writes are complete.
// Saves about two microseconds between the kernels of one call.  What the kernel before it writes is taken by plain pointers:
// behind `const ... __restrict__` the compiler may use loads that demand memory which nobody writes while the kernel lives, and
// may move them before the wait.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute behind[1];
    behind[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    behind[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = dim3(threads), config.dynamicSmemBytes = smem, config.stream = st;
    config.attrs = behind, config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, P(args)...);
}

// ---- arguments -------------------------------------------------------------------------------

// 0 for a value that names no type
inline size_t type_bytes(alphasparse_cuda_type_t t) {
    return t == ALPHA_SPARSE_CUDA_TYPE_F32 ? 4 : t == ALPHA_SPARSE_CUDA_TYPE_F16 || t == ALPHA_SPARSE_CUDA_TYPE_BF16 ? 2 : 0;
}
inline size_t index_bytes(alphasparse_cuda_index_t t) {
    return t == ALPHA_SPARSE_CUDA_INDEX_I32 ? 4 : t == ALPHA_SPARSE_CUDA_INDEX_I64 ? 8 : 0;
}

constexpr int64_t kMostRows = 0x7fffffff - 4096;  // row counts and positions fit an int with room for a tile's overhang
constexpr int64_t kMostWidth = 1 << 24;
constexpr int64_t kMostStride = 0x7fffffff;
constexpr int kMostExperts = 1024;
constexpr int kMostTopK = 32;

// One operand: `rows` rows of `width` elements of `elem` bytes, `ld` elements apart.
struct Operand {
    const void *p;
    int64_t rows, width, ld;
    size_t elem;
    bool written;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t end() const {
        return begin() + (rows > 0 ? (((uintptr_t)rows - 1) * (uintptr_t)ld + (uintptr_t)width) * elem : 0);
    }
    bool empty() const { return rows <= 0 || width <= 0; }
};

// Checks operands in the order that they are given: there (NOT_INITIALIZED), leading dimension and alignment to the
// element (INVALID_VALUE), no written operand in the place of another (INVALID_VALUE; columns of one block of rows beside each
// other are two places), memory of the current device
// (INVALID_POINTER).  Operands without elements may be null.  An optional operand is left out by the caller.
alphasparse_status_t check_operands(const char *call, std::initializer_list<Operand> operands);

// Largest of 16, 8, 4 and the element's own bytes that divides everything given (addresses, strides and widths in bytes).
inline int vector_bytes(size_t elem, std::initializer_list<uint64_t> all) {
    uint64_t any = 0;
    for (uint64_t v : all) any |= v;
    return any % 16 == 0 ? 16 : any % 8 == 0 ? 8 : any % 4 == 0 ? 4 : (int)elem;
}

inline uint64_t address(const void *p) { return (uint64_t)reinterpret_cast<uintptr_t>(p); }

constexpr int kRowThreads = 256;

// log2 of the threads, at most a block, that share a row of `nv` vectors, `unroll` vectors a thread at a time.  Few vectors in
// all: as many as the row has, so that it is done in one round trip to memory.  Many: the number from 2^least up that leaves the
// fewest of them idle in the row's last piece, the largest of equals.  (Rows of 272 vectors, by a whole block twice: combine 55 us,
// its gradient 104; by 32 and 64 threads 47 and 78.)  Wide rows in groups of a warp or more; rows of up to 1 KB in groups
// from 8 threads on (33 vectors: 20 us, 27 by warps).
inline int row_group(int64_t rows, int64_t nv, int unroll, int least) {
    int best = 0;
    while ((1 << best) < kRowThreads && (int64_t)unroll << best < nv) best++;
    if (rows * nv <= 148 * 2048 || nv > 16 * (int64_t)unroll * kRowThreads) return best;  // of many pieces, one more or less
    const auto slots = [&](int log) {
        const int64_t piece = (int64_t)unroll << log;
        return (nv + piece - 1) / piece * piece;
    };
    for (int log = best - 1; log >= least; log--)
        if (slots(log) < slots(best)) best = log;
    return best;
}

// A row by groups of 2^log threads, `unroll` vectors a thread and piece of the row: one where there are few in all; many: `many`,
// so that enough are in flight.
struct RowShape {
    int log, unroll;
    dim3 grid;
};
inline RowShape row_shape(int64_t rows, int64_t nv, int many, int least) {
    RowShape s;
    s.unroll = rows * nv <= 148 * 2048 ? 1 : many;
    s.log = row_group(rows, nv, s.unroll, least);
    const int64_t per_block = kRowThreads >> s.log, piece = (int64_t)s.unroll << s.log;
    s.grid = dim3((unsigned)((rows + per_block - 1) / per_block), (unsigned)((nv + piece - 1) / piece));
    return s;
}

inline Window window(const void *p, int64_t rows, int64_t width, int64_t ld, size_t elem) {
    const char *lo = static_cast<const char *>(p);
    return Window{lo, lo + (rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)width) * elem : 0)};
}

}  // namespace asb

// Calls f with a value of the element type that `type` names
#define ASB_BY_TYPE(type, f)                                                     \
    switch (type) {                                                              \
        case ALPHA_SPARSE_CUDA_TYPE_F32: f((float)0); break;                     \
        case ALPHA_SPARSE_CUDA_TYPE_F16: f(__half()); break;                     \
        case ALPHA_SPARSE_CUDA_TYPE_BF16: f(__nv_bfloat16()); break;             \
    }
