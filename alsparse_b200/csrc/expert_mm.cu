// Products of the experts: rows [offsets[e], offsets[e + 1]) of a dense block times the weights of expert e (a block-diagonal
// matrix times a dense block), and the gradient of the weights.  No counterpart in the reference.
//
// expert_mm_kernel: tcgen05.mma with operands brought by TMA into a ring of stages, accumulators in TMEM, persistent blocks,
// one per SM.  One warp issues copies, one the products, eight empty the accumulators; two accumulators, so that a tile is
// written while the next is multiplied.  The rows of an expert are the narrow side of the tile: its width is any multiple
// of 16, so an expert's rows are cut into equal tiles of at most 256, and no more rows are fetched and written than there
// are.  (64 of k take 233 ns at n = 16, 304 at 256: the four products take 270 at 256, and
// what there is to do around them is no less with narrow ones.  So a narrow tile of weights streams at most 70 GB/s through an SM.)  With many rows an expert two SMs work on one tile of
// 256 (cta_group::2), which halves what each fetches of the narrow operand.  The offsets stay on the device: every block
// forms the same table of row tiles.
// Addresses or strides that TMA does not take (no multiple of 16 bytes) are brought by fourteen warps of their own instead.
// expert_mm_plain_kernel: 32-bit operands, on the ordinary units (4096 rows of 16 experts, 1024 x 1024: 345 us forward, 25 TFLOP/s,
// gradient 298 us); and what 16-bit calls leave when there is nothing to sum, no rows or sums of length zero.
#include <cuda.h>
#include <stdio.h>

#include <algorithm>

#include "expert_tiles.h"
#include "rows.h"

namespace asb {

// Set by a kernel whose bounded wait ran out (alphasparse_cuda_expert_mm_status).
static __device__ int g_expert_mm_status;
// What a call to it reads.  Read and cleared in one step, so that no failure falls between the two.
static __device__ int g_expert_mm_told;
static __global__ void tell_status_kernel(int clear) {
    g_expert_mm_told = clear ? atomicExch(&g_expert_mm_status, 0) : atomicAdd(&g_expert_mm_status, 0);
}

// D[m, n] = sum over k of A[m, k] B[n, k].  What the three dimensions are:
enum MmForm {
    kRows,     // m: output features, n: rows of an expert, k: input features
    kGradient  // m: columns of x, n: columns of dy, k: rows of an expert   (dW^T = x^T dy)
};

// First and last row of an expert, whatever the offsets hold
__device__ __forceinline__ void rows_of(const int *__restrict__ offsets, int e, int64_t rows, int *lo, int *hi) {
    const int64_t a = min(max((int64_t)__ldg(offsets + e), (int64_t)0), rows);
    *lo = (int)a;
    *hi = (int)min(max((int64_t)__ldg(offsets + e + 1), a), rows);
}

// begin[e] = offsets[e] within [0, rows], for the whole block to read after a barrier; whoever reads it takes an expert whose end lies
// before its begin for one without rows
__device__ __forceinline__ void load_offsets(const int *__restrict__ offsets, int experts, int64_t rows, int *begin) {
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) begin[e] = (int)min(max((int64_t)__ldg(offsets + e), (int64_t)0), rows);
}

// first[e] = row tiles of the experts before e, e = 0 .. experts; by one warp, from begin.  Offsets that name more rows than
// there are (they do not ascend) give no tiles at all.
__device__ __forceinline__ void count_row_tiles(const int *begin, int experts, int64_t rows, int tile, int *first) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
    int64_t named = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
        const int e = e0 + lane, here = e < experts ? max(0, begin[e + 1] - begin[e]) : 0;
        const int n = (here + tile - 1) / tile;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        // the sum of 32 counts may pass an int
        named += (int64_t)__reduce_add_sync(0xffffffffu, (unsigned)here >> 16) * 65536 + __reduce_add_sync(0xffffffffu, (unsigned)here & 0xffffu);
        if (named > rows) {
            carry = 0;
            break;
        }
        if (e < experts) first[e] = carry + inc - n;
        carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) first[experts] = carry;
}

// the expert of row tile r
__device__ __forceinline__ int expert_of(const int *first, int experts, int r) {
    int lo = 0, hi = experts - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- without tensor cores ------------------------------------------------------------------------

constexpr int kPlainTile = 64, kPlainStep = 16;

// One block per tile of 64 x 64, a thread 4 x 4 of it.  AK / BK: consecutive k are consecutive in memory.
template <typename T, typename TO, bool GRAD, bool AK, bool BK>
__global__ void __launch_bounds__(256)
    expert_mm_plain_kernel(const int *__restrict__ offsets, int experts, int64_t rows, int m_size, int n_size, int k_size,
                           const T *__restrict__ a, int64_t lda, int64_t stride_a, const T *__restrict__ b, int64_t ldb,
                           int64_t stride_b, float beta, TO *__restrict__ c, int64_t ldc, int64_t stride_c) {
    __shared__ int s_first[kMostExperts + 1], s_begin[kMostExperts + 1];
    __shared__ __align__(16) float s_a[kPlainStep][kPlainTile + 4], s_b[kPlainStep][kPlainTile + 4];  // read four at a time
    int e, lo, hi, m0, m_end, k_end;
    int n0 = blockIdx.x * kPlainTile;
    if (GRAD) {  // the tiles of an expert along x, both ways
        e = blockIdx.z;
        rows_of(offsets, e, rows, &lo, &hi);
        const unsigned across = ((unsigned)n_size + kPlainTile - 1) / kPlainTile, down = blockIdx.x / across;
        n0 = (int)(blockIdx.x - down * across) * kPlainTile;
        m0 = (int)down * kPlainTile, m_end = m_size, k_end = hi - lo;
    } else {
        load_offsets(offsets, experts, rows, s_begin);
        __syncthreads();
        if (threadIdx.x < 32) count_row_tiles(s_begin, experts, rows, kPlainTile, s_first);
        __syncthreads();
        const int r = (int)(blockIdx.y + blockIdx.z * gridDim.y);
        if (r >= s_first[experts]) return;
        e = expert_of(s_first, experts, r);
        rows_of(offsets, e, rows, &lo, &hi);
        m0 = (r - s_first[e]) * kPlainTile, m_end = hi - lo, k_end = k_size;
    }
    // the operand that is indexed by rows begins at the expert's first
    const T *pa = a + lo * lda + e * stride_a;
    const T *pb = b + (GRAD ? lo * ldb : 0) + e * stride_b;
    float acc[4][4] = {};
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int k0 = 0; k0 < k_end; k0 += kPlainStep) {
#pragma unroll
        for (int i = threadIdx.x; i < kPlainTile * kPlainStep; i += 256) {
            const int am = AK ? i / kPlainStep : i % kPlainTile, ak = AK ? i % kPlainStep : i / kPlainTile;
            s_a[ak][am] = m0 + am < m_end && k0 + ak < k_end ? to_float(AK ? pa[(int64_t)(m0 + am) * lda + k0 + ak] : pa[(int64_t)(k0 + ak) * lda + m0 + am]) : 0.f;
            const int bn = BK ? i / kPlainStep : i % kPlainTile, bk = BK ? i % kPlainStep : i / kPlainTile;
            s_b[bk][bn] = n0 + bn < n_size && k0 + bk < k_end ? to_float(BK ? pb[(int64_t)(n0 + bn) * ldb + k0 + bk] : pb[(int64_t)(k0 + bk) * ldb + n0 + bn]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPlainStep; k++) {
            const float4 va = *reinterpret_cast<const float4 *>(&s_a[k][ty * 4]), vb = *reinterpret_cast<const float4 *>(&s_b[k][tx * 4]);
            const float fa[4] = {va.x, va.y, va.z, va.w}, fb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int m = m0 + ty * 4 + i;
        if (m >= m_end) continue;
        TO *row = c + (GRAD ? e * stride_c + m * ldc : (int64_t)(lo + m) * ldc);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = n0 + tx * 4 + j;
            if (n < n_size) row[n] = from_float<TO>(beta != 0.f ? fmaf(beta, to_float(row[n]), acc[i][j]) : acc[i][j]);
        }
    }
}

// ---- tensor cores --------------------------------------------------------------------------------

constexpr int kMmThreads = 384;  // copies, products, eight warps for the accumulators, two for the ends of ragged experts
constexpr int kMmCopyWarps = 14;  // ANY: after the others, instead of the two for ragged ends
constexpr int kMmThreadsAny = 320 + 32 * kMmCopyWarps;
constexpr int kMmM = 128, kMmK = 64;

__device__ __forceinline__ unsigned smem_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint64_t *b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_address(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_address(b)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(b)), "r"(bytes) : "memory");
}
// True in one lane of a converged warp, always the same one.  The copies and products are issued under this and not under a
// test of the lane's number: the compiler then keeps their operands in uniform registers (as it is, a product of
// 128 x 32 x 16 was issued every 250 cycles under lane == 0).  What the warp of the products does for 64 of k besides bounds
// narrow tiles: 273 ns with an election each time, 233 ns with one lane for the whole loop and the four products written out.
// The copying warp is better off with all lanes in the loop (one lane: 249 to 303 ns).
__device__ __forceinline__ bool elect_one() {
    unsigned one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of the given parity; false when it ran out of time or another thread of the block did.  `work`: what the
// block may have to do first (tile_work).  CLUSTER: what the pair's other block wrote before it arrived is seen (dear: about a
// microsecond).
template <bool CLUSTER = false>
__device__ __forceinline__ bool barrier_wait(uint64_t *b, unsigned parity, volatile int *s_stop, long long work) {
    unsigned long long begin = 0;
    for (unsigned i = 0;; i++) {
        unsigned done;
        if constexpr (CLUSTER)
            asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                         : "=r"(done)
                         : "r"(smem_address(b)), "r"(parity)
                         : "memory");
        else
            asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                         : "=r"(done)
                         : "r"(smem_address(b)), "r"(parity)
                         : "memory");
        if (done) return true;
        if ((i & 15) == 15) {
            if (*s_stop) return false;
            const unsigned long long t = now_ns();
            if (!begin) begin = t;
            else if (t - begin > wait_limit_ns(work)) {
                *s_stop = 1;
                return false;
            }
        }
    }
}
// ... by a whole warp, with one answer for all lanes
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t *b, unsigned parity, volatile int *s_stop, long long work) {
    return __all_sync(0xffffffffu, barrier_wait<CLUSTER>(b, parity, s_stop, work));
}
// After the last copy: waits until every stage has been used for the last time, so that no arrival of a product comes to a block
// that has ended (the products' arrivals on two barriers need not come in their order).  A stage that was never filled is free.
__device__ __forceinline__ void last_uses(uint64_t *empty, int stage, unsigned phase, int stages, volatile int *s_stop, long long work) {
    for (int i = 0; i < stages; i++) {
        if (!warp_wait(&empty[stage], phase ^ 1, s_stop, work)) return;
        if (++stage == stages) stage = 0, phase ^= 1;
    }
}
// PAIR: `barrier` is an address of the cluster's, the other block's too
template <bool PAIR>
__device__ __forceinline__ void copy_tile(void *dst, const CUtensorMap *map, int x, int y, int z, unsigned barrier) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         smem_address(dst)),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(barrier)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         smem_address(dst)),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(barrier)
                     : "memory");
}
// Shared-memory descriptor of an operand whose rows are 128 bytes, swizzled by 128 bytes.  K-major: rows of 64 k, groups of
// eight rows 1024 bytes apart.  M/N-major: rows of 64 m (or n) per k, groups of eight k 1024 bytes apart, and the next 64 m
// 8192 bytes on (a box of 64 k).
__device__ __forceinline__ uint64_t operand_descriptor(unsigned address, bool k_major) {
    return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)(k_major ? 1 : 8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool PAIR>
__device__ __forceinline__ void multiply(unsigned d, uint64_t a, uint64_t b, unsigned instruction, bool add) {
    if constexpr (PAIR)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(instruction), "r"((unsigned)add)
                     : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(instruction), "r"((unsigned)add)
                     : "memory");
}
// An arrival on the barrier (PAIR: on that of both blocks) when the products issued so far are done
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *b) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_address(b)),
                     "h"((unsigned short)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(b)) : "memory");
}
// The address, in the cluster's window, that `p` has in the pair's first block
__device__ __forceinline__ unsigned address_in_first(const void *p) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_address(p)));
    return a;
}
// An arrival on the barrier of the pair's first block.  RELEASE: with what this thread wrote to memory before
template <bool RELEASE>
__device__ __forceinline__ void arrive_at_first(uint64_t *b) {
    if constexpr (RELEASE) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(address_in_first(b)) : "memory");
    else asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(address_in_first(b)) : "memory");
}
__device__ __forceinline__ void pair_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Requests 32 columns of this warp's 32 lanes; they are there after wait_accumulators.
__device__ __forceinline__ void request_accumulators(unsigned address, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address)
        : "memory");
}
// The registers are named so that no use of them is moved before the wait.
__device__ __forceinline__ void wait_accumulators(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// A warp writes a block of 32 rows x 32 columns of the output: a lane has one column, its register i row i.  dst: row 0, the
// warp's first column; `rows` and `cols` of them exist.  32-bit elements: a row is a line, as it is.  16-bit ones are
// exchanged among eight lanes in three steps, until a lane has eight columns of four rows and writes 16 bytes at a time (a
// store of two bytes a lane and row took 923 us where this takes 705 us: 32,768 rows of 8 experts, 4096 x 4096,
// operation N).
template <typename TO>
__device__ __forceinline__ void write_block(const unsigned (&r)[32], TO *dst, int64_t ldo, int rows, int cols, bool vectors, float beta) {
    const int lane = threadIdx.x & 31;
    if constexpr (sizeof(TO) == 2) {
        if (vectors && beta == 0.f) {
            unsigned p[16];
            const unsigned halves = lane & 1 ? 0x3276 : 0x5410;  // the odd rows of both lanes, or the even ones
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const unsigned own = pack_two<TO>(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                p[i] = __byte_perm(own, __shfl_xor_sync(0xffffffffu, own, 1), halves);
            }
            const bool second = lane & 2, upper = lane & 4;
            uint2 h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const unsigned other = __shfl_xor_sync(0xffffffffu, second ? p[2 * i] : p[2 * i + 1], 2);
                h[i] = make_uint2(second ? other : p[2 * i], second ? p[2 * i + 1] : other);
            }
            const int first = lane & ~7;
            TO *to = dst + (lane & 7) * ldo + first;
            const bool whole = rows >= 32 && cols >= 32;
#pragma unroll
            for (int i = 0; i < 4; i++, to += 8 * ldo) {
                const unsigned ox = __shfl_xor_sync(0xffffffffu, upper ? h[2 * i].x : h[2 * i + 1].x, 4);
                const unsigned oy = __shfl_xor_sync(0xffffffffu, upper ? h[2 * i].y : h[2 * i + 1].y, 4);
                const uint4 o = make_uint4(upper ? ox : h[2 * i].x, upper ? oy : h[2 * i].y, upper ? h[2 * i + 1].x : ox, upper ? h[2 * i + 1].y : oy);
                if (whole || (8 * i + (lane & 7) < rows && first + 8 <= cols)) {
                    *reinterpret_cast<uint4 *>(to) = o;
                } else if (8 * i + (lane & 7) < rows) {
                    const unsigned e[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (first + j < cols) reinterpret_cast<unsigned short *>(to)[j] = (unsigned short)(e[j / 2] >> 16 * (j & 1));
                }
            }
            return;
        }
    }
    if (lane >= cols) return;
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (i < rows) {
            TO *to = dst + i * ldo + lane;
            const float v = __uint_as_float(r[i]);
            *to = from_float<TO>(beta != 0.f ? fmaf(beta, to_float(*to), v) : v);
        }
}

struct MmShape {
    const int *offsets;
    int experts;
    int64_t rows;
    int m_size;        // kRows: columns of the output (features); kGradient: columns of x
    int n_size;        // kGradient: columns of dy
    int reduced;       // kRows: length of the sum
    int n, stages;     // widest tile, depth of the ring
    int m_tiles, n_tiles;
    unsigned stage_bytes, instruction, acc_stride;
    bool vectors;      // rows of the output begin on 16-byte boundaries
    float beta;
    // ANY: the operands themselves (a: the weights of all experts, or x; b: x, or dy)
    const void *a, *b;
    int64_t lda, ldb, stride_a;
    Window all_a, all_b;
};

// ANY: a thread's share of an operand's part of a stage, in the order that the copies of TMA leave it in (16 bytes c of a row of
// 128 bytes at c ^ (row & 7)).  K_MAJOR: one box of `extent` rows; else boxes of 64 rows side by side, `extent` columns wide.  Only
// `rows_there` rows and `cols_there` columns exist; the rest becomes zeros.
template <typename T, bool K_MAJOR>
__device__ __forceinline__ void copy_boxes(char *dst, const T *src, int64_t ld, const Window &all, int extent, int rows_there,
                                           int cols_there, int thread) {
    constexpr int E = 16 / sizeof(T), ahead = 3;  // chunks a thread has on their way
    const int chunks = K_MAJOR ? extent * 8 : (extent + 63) / 64 * 512;
    for (int i0 = thread; i0 < chunks; i0 += ahead * 32 * kMmCopyWarps) {
        AnyPack<T> p[ahead];
#pragma unroll
        for (int u = 0; u < ahead; u++) {
            const int i = i0 + u * 32 * kMmCopyWarps, row = K_MAJOR ? i >> 3 : i >> 3 & 63, col = (K_MAJOR ? 0 : i >> 9) * 64 + (i & 7) * E;
            p[u] = AnyPack<T>(src + row * ld + col, all, i < chunks && row < rows_there && col + E <= cols_there);
        }
#pragma unroll
        for (int u = 0; u < ahead; u++) {
            const int i = i0 + u * 32 * kMmCopyWarps, row = K_MAJOR ? i >> 3 : i >> 3 & 63, col = (K_MAJOR ? 0 : i >> 9) * 64 + (i & 7) * E;
            if (i >= chunks) break;
            Pack<T, E> v = p[u].get();
            if (row < rows_there && col < cols_there && col + E > cols_there) {
                float f[E];
#pragma unroll
                for (int j = 0; j < E; j++) f[j] = col + j < cols_there ? to_float(__ldg(src + row * ld + col + j)) : 0.f;
                v = pack<T, E>(f);
            }
            // rows of all boxes are 128 bytes apart
            store_pack<T, E>(reinterpret_cast<T *>(dst + (i >> 3) * 128 + (((i & 7) ^ (i >> 3 & 7)) << 4)), v);
        }
    }
}

struct MmTile {
    int expert, m0, n0, n;  // n0: first row (kRows) or column of dy; n: width of the product, a multiple of 16 (two blocks: 32)
    int lo, length;         // kGradient: the expert's first row, its rows; kRows: length = rows of the tile
    int steps;
};

template <int FORM, bool PAIR>
__device__ __forceinline__ MmTile mm_tile(const MmShape &s, const int *s_first, const int *s_begin, int t) {
    constexpr int M = PAIR ? 2 * kMmM : kMmM, unit = PAIR ? 32 : 16;
    MmTile q;
    int hi;
    if (FORM == kGradient) {
        const int per = s.m_tiles * s.n_tiles;
        q.expert = t / per;
        const int i = t - q.expert * per, f = i / s.n_tiles;
        q.lo = s_begin[q.expert], hi = max(q.lo, s_begin[q.expert + 1]);
        q.m0 = f * M, q.n0 = (i - f * s.n_tiles) * s.n;
        q.n = min(s.n, (s.n_size - q.n0 + unit - 1) / unit * unit);
        q.length = hi - q.lo;
        q.steps = (q.length + kMmK - 1) / kMmK;
    } else {
        const int r = t / s.m_tiles, f = t - r * s.m_tiles;
        q.expert = expert_of(s_first, s.experts, r);
        q.lo = s_begin[q.expert], hi = max(q.lo, s_begin[q.expert + 1]);
        // equal shares of the expert's rows
        const int share = equal_share(hi - q.lo, s_first[q.expert + 1] - s_first[q.expert], unit);
        q.n0 = q.lo + (r - s_first[q.expert]) * share;
        q.length = min(share, hi - q.n0);
        q.n = (q.length + unit - 1) / unit * unit;
        q.m0 = f * M;
        q.steps = (s.reduced + kMmK - 1) / kMmK;
    }
    return q;
}

// kGradient: step k ends within a group of 16 rows, the unit of the products
__device__ __forceinline__ bool ragged(const MmTile &q, int k) { return q.length - k * kMmK < kMmK && (q.length & 15) != 0; }

// W_K: consecutive terms of the sums are consecutive in memory (K-major weights), else consecutive features.  PAIR: two blocks
// of a cluster on one tile: each fetches its 128 of the 256 m and its half of n, the first issues the products of both, the
// accumulators of a block's 128 m are its own.  The copies of both report to the first block's barrier, but for the
// last rows of an expert in kGradient: each block waits for its own and clears what does not belong to the expert (its last
// warp), and tells the first.
template <int FORM, bool PAIR, bool W_K, bool ANY, typename T, typename TO>
__global__ void __launch_bounds__(ANY ? kMmThreadsAny : kMmThreads, 1)
    expert_mm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_c, const MmShape s,
                     TO *__restrict__ out, int64_t ldo, int64_t stride_o) {
    constexpr bool a_k = FORM == kRows && W_K, b_k = FORM == kRows;
    constexpr unsigned a_bytes = kMmM * kMmK * sizeof(T);
    extern __shared__ __align__(16) char s_raw[];
    __shared__ int s_first[kMostExperts + 1], s_begin[kMostExperts + 1];  // row tiles before an expert; the offsets, clamped
    __shared__ uint64_t s_full[kMmMostStages], s_empty[kMmMostStages], s_own[2 * kMmMostStages], s_ready[kMmMostStages], s_acc_full[2], s_acc_empty[2];
    __shared__ unsigned s_tmem;
    __shared__ int s_stop_word;
    volatile int *s_stop = &s_stop_word;
    char *ring = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    const int w = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // clusters of two along x
    const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
    constexpr unsigned columns = 512;  // all of TMEM: one block per SM

    load_offsets(s.offsets, s.experts, s.rows, s_begin);
    if (w == 0) {
        if (lane == 0) {
            if (!ANY) {
                asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
                if (b_k) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c) : "memory");
            }
            for (int i = 0; i < s.stages; i++) barrier_init(&s_full[i], ANY ? kMmCopyWarps : 1), barrier_init(&s_empty[i], 1), barrier_init(&s_ready[i], PAIR ? 2 : 1);
            for (int i = 0; i < 2 * kMmMostStages; i++) barrier_init(&s_own[i], 1);
            for (int i = 0; i < 2; i++) barrier_init(&s_acc_full[i], 1), barrier_init(&s_acc_empty[i], PAIR ? 16 : 8);
            s_stop_word = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    } else if (w == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&s_tmem)), "r"(columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&s_tmem)), "r"(columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (FORM == kRows) {
        if (w == 2) count_row_tiles(s_begin, s.experts, s.rows, s.n, s_first);
        __syncthreads();
    }
    if constexpr (PAIR) pair_barrier();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = s_tmem;
    const int tiles = FORM == kGradient ? s.experts * s.m_tiles * s.n_tiles : s_first[s.experts] * s.m_tiles;
    long long work = 0;  // of this warp's tiles so far, for the limits of its waits

    if (w == 0) {
        int stage = 0;
        unsigned phase = 0;
        EndTurn turn;
        bool good = !ANY;
        for (int t = worker; good && t < tiles; t += workers) {
            const MmTile q = mm_tile<FORM, PAIR>(s, s_first, s_begin, t);
            work += tile_work(q.steps);
            const int half = PAIR ? q.n >> 1 : q.n, m0 = q.m0 + rank * kMmM, n0 = q.n0 + rank * half;
            // kRows: boxes of 64 rows, then of 16; kGradient: boxes of 64 columns
            const int wide = b_k ? half >> 6 : (half + 63) >> 6, narrow = b_k ? (half & 63) >> 4 : 0;
            const unsigned bytes = a_bytes + (unsigned)wide * 8192u + (unsigned)narrow * 2048u;
            for (int k = 0; k < q.steps; k++) {
                if (!(good = warp_wait(&s_empty[stage], phase ^ 1, s_stop, work))) break;
                char *a = ring + (size_t)stage * s.stage_bytes, *b = a + a_bytes;
                const int k0 = k * kMmK;
                const auto copy = [&](auto both, unsigned barrier) {
                    constexpr bool B = decltype(both)::value;
                    if (a_k) copy_tile<B>(a, &map_a, k0, m0, q.expert, barrier);
                    else
                        for (int g = 0; g < kMmM / 64; g++)
                            copy_tile<B>(a + g * 8192, &map_a, m0 + g * 64, FORM == kGradient ? q.lo + k0 : k0, FORM == kGradient ? 0 : q.expert, barrier);
                    for (int g = 0; g < wide; g++) {
                        if (b_k) copy_tile<B>(b + g * 8192, &map_b, k0, n0 + g * 64, 0, barrier);
                        else copy_tile<B>(b + g * 8192, &map_b, n0 + g * 64, q.lo + k0, 0, barrier);
                    }
                    for (int g = 0; g < narrow; g++) copy_tile<B>(b + wide * 8192 + g * 2048, &map_c, k0, n0 + wide * 64 + g * 16, 0, barrier);
                };
                const bool end = !ANY && FORM == kGradient && ragged(q, k);
                uint64_t *own = &s_own[end ? end_barrier(turn.take(), stage) : 0];
                if (elect_one()) {
                    if (end) {
                        barrier_expect(own, bytes);
                        copy(std::false_type{}, smem_address(own));
                    } else if (PAIR) {
                        if (rank == 0) barrier_expect(&s_full[stage], 2 * bytes);
                        copy(std::true_type{}, address_in_first(&s_full[stage]));
                    } else {
                        barrier_expect(&s_full[stage], bytes);
                        copy(std::false_type{}, smem_address(&s_full[stage]));
                    }
                }
                __syncwarp();
                if (++stage == s.stages) stage = 0, phase ^= 1;
            }
        }
        if (good) last_uses(s_empty, stage, phase, s.stages, s_stop, work);
    } else if (w == 1 && rank == 0 && elect_one()) {
        int stage = 0, count = 0;
        unsigned full_phases = 0, ready_phases = 0;  // a bit for each stage: the phase that comes next
        bool good = true;
        for (int t = worker; good && t < tiles; t += workers) {
            const MmTile q = mm_tile<FORM, PAIR>(s, s_first, s_begin, t);
            work += tile_work(q.steps);
            if (q.steps == 0) continue;
            const int slot = count & 1;
            if (!(good = barrier_wait(&s_acc_empty[slot], ((count >> 1) & 1) ^ 1, s_stop, work))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            count++;
            const int length = FORM == kGradient ? q.length : s.reduced;
            const unsigned instruction = s.instruction | (unsigned)(q.n >> 3) << 17;
            const unsigned d = tmem + slot * s.acc_stride;
            for (int k = 0; k < q.steps; k++) {
                char *a = ring + (size_t)stage * s.stage_bytes;
                const int left = length - k * kMmK, parts = min(4, (left + 15) / 16);
                if (!ANY && FORM == kGradient && ragged(q, k)) {
                    if (!(good = barrier_wait<true>(&s_ready[stage], ready_phases >> stage & 1, s_stop, work))) break;
                    ready_phases ^= 1u << stage;
                } else {
                    if (!(good = barrier_wait(&s_full[stage], full_phases >> stage & 1, s_stop, work))) break;
                    full_phases ^= 1u << stage;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t da = operand_descriptor(smem_address(a), a_k), db = operand_descriptor(smem_address(a + a_bytes), b_k);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (i < parts)
                        multiply<PAIR>(d, da + (uint64_t)(i * (a_k ? 32 : 2048) >> 4), db + (uint64_t)(i * (b_k ? 32 : 2048) >> 4), instruction,
                                       k > 0 || i > 0);
                commit<PAIR>(&s_empty[stage]);
                if (k == q.steps - 1) commit<PAIR>(&s_acc_full[slot]);
                if (++stage == s.stages) stage = 0;
            }
        }
    } else if (w >= 2 && w < 10) {
        // the quarter of the accumulators' lanes that this warp may read, and whether it takes the even or the odd blocks of 32
        // columns (four warps alone take longer for a tile than the products of a few hundred rows)
        const int part = w & 3, odd = (w - 2) >> 2;
        int count = 0;
        for (int t = worker; t < tiles; t += workers) {
            const MmTile q = mm_tile<FORM, PAIR>(s, s_first, s_begin, t);
            work += tile_work(q.steps);
            const int slot = count & 1, m = q.m0 + rank * kMmM + part * 32;
            if (q.steps > 0) {
                if (!warp_wait(&s_acc_full[slot], (count >> 1) & 1, s_stop, work)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                count++;
            }
            const unsigned from = tmem + slot * s.acc_stride + ((unsigned)(part * 32) << 16);
            const int rows = FORM == kGradient ? min(q.n, s.n_size - q.n0) : q.length;
            TO *dst = out + (FORM == kGradient ? q.expert * stride_o : 0) + (int64_t)q.n0 * ldo + m;
            if (q.steps == 0) {
                // an expert without rows: beta times what is there, a row of the block's 128 columns per warp and step
                TO *all = dst - part * 32;
                const int cols = min(kMmM, s.m_size - q.m0 - rank * kMmM);
                for (int r = w - 2; r < rows; r += 8) {
                    TO *to = all + r * ldo;
                    if (s.vectors && s.beta == 0.f && cols == kMmM) {
                        if (lane * 16 < kMmM * (int)sizeof(TO)) reinterpret_cast<uint4 *>(to)[lane] = make_uint4(0, 0, 0, 0);
                    } else {
                        for (int c = lane; c < cols; c += 32) to[c] = from_float<TO>(s.beta != 0.f ? s.beta * to_float(to[c]) : 0.f);
                    }
                }
            } else if (m < s.m_size) {
                for (int c = odd * 32; c < rows; c += 64) {
                    unsigned v[32];
                    request_accumulators(from + c, v);
                    wait_accumulators(v);
                    write_block<TO>(v, dst + c * ldo, ldo, rows - c, s.m_size - m, s.vectors, s.beta);
                }
            }
            if (q.steps > 0) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) arrive_at_first<false>(&s_acc_empty[slot]);
                    else barrier_arrive(&s_acc_empty[slot]);
                }
            }
        }
    } else if (ANY && w >= 10) {
        const int thread = threadIdx.x - 320;
        int stage = 0;
        unsigned phase = 0;
        bool good = true;
        for (int t = worker; good && t < tiles; t += workers) {
            const MmTile q = mm_tile<FORM, PAIR>(s, s_first, s_begin, t);
            work += tile_work(q.steps);
            for (int k = 0; k < q.steps; k++) {
                if (!(good = warp_wait(&s_empty[stage], phase ^ 1, s_stop, work))) break;
                char *a = ring + (size_t)stage * s.stage_bytes, *b = a + a_bytes;
                const int k0 = k * kMmK, m_there = s.m_size - q.m0;
                const T *pa = static_cast<const T *>(s.a), *pb = static_cast<const T *>(s.b);
                if (FORM == kGradient) {
                    const int there = q.length - k0;
                    copy_boxes<T, false>(a, pa + (int64_t)(q.lo + k0) * s.lda + q.m0, s.lda, s.all_a, kMmM, there, m_there, thread);
                    copy_boxes<T, false>(b, pb + (int64_t)(q.lo + k0) * s.ldb + q.n0, s.ldb, s.all_b, q.n, there, s.n_size - q.n0, thread);
                } else {
                    const int there = s.reduced - k0;
                    pa += q.expert * s.stride_a;
                    if (W_K) copy_boxes<T, true>(a, pa + (int64_t)q.m0 * s.lda + k0, s.lda, s.all_a, kMmM, m_there, there, thread);
                    else copy_boxes<T, false>(a, pa + (int64_t)k0 * s.lda + q.m0, s.lda, s.all_a, kMmM, there, m_there, thread);
                    copy_boxes<T, true>(b, pb + (int64_t)q.n0 * s.ldb + k0, s.ldb, s.all_b, q.n, q.length, there, thread);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) barrier_arrive(&s_full[stage]);
                if (++stage == s.stages) stage = 0, phase ^= 1;
            }
        }
        if (good) last_uses(s_empty, stage, phase, s.stages, s_stop, work);
    } else if (FORM == kGradient && w >= 10) {
        // the ends of experts whose rows are no multiple of 16: rows of the next expert (or behind the last) came along with
        // the copy.  Zeros in both operands up to the next multiple, so that nothing that stands there, NaN included, gets
        // into the sum; then the first block's products may go on.  Two warps in turn: one alone takes 1.7 us a tile, of which its
        // fence and arrival are most, and the rest of a short tile 1.0.
        int stage = 0;
        unsigned own_phases = 0;  // a bit for each stage: the phase that comes next
        EndTurn turn;
        bool good = true;
        for (int t = worker; good && t < tiles; t += workers) {
            const MmTile q = mm_tile<FORM, PAIR>(s, s_first, s_begin, t);
            work += tile_work(q.steps);
            const int last = q.steps - 1, left = q.length - last * kMmK;
            if (q.steps > 0 && ragged(q, last)) {
                const int at = (stage + last) % s.stages;
                if (turn.take() == (w & 1)) {
                    if (!(good = warp_wait(&s_own[end_barrier(w & 1, at)], own_phases >> at & 1, s_stop, work))) break;
                    own_phases ^= 1u << at;
                    char *a = ring + (size_t)at * s.stage_bytes;
                    const int end = ((left + 15) / 16 * 16 - left) * 8, boxes = 2 + (((PAIR ? q.n >> 1 : q.n) + 63) >> 6);
                    for (int box = 0; box < boxes; box++)
                        for (int i = lane; i < end; i += 32)
                            *reinterpret_cast<uint4 *>(a + (size_t)box * 8192 + left * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive_at_first<true>(&s_ready[at]);
                }
            }
            stage = (stage + q.steps) % s.stages;
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*s_stop) {
        // a wait ran out: what is still on its way into shared memory gets time to arrive before the block goes
        if (threadIdx.x == 0) {
            atomicExch(&g_expert_mm_status, 1);
            const unsigned long long begin = now_ns();
            while (now_ns() - begin < 10000000ull) __nanosleep(1000);
        }
        __syncthreads();
    }
    if constexpr (PAIR) pair_barrier();  // nothing reaches into the other block's memory after this
    if (w == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static std::atomic<void *> known{nullptr};  // once it was found
    void *p = known.load();
    if (p) return reinterpret_cast<EncodeTiled>(p);
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
        return nullptr;
    known.store(p);
    return reinterpret_cast<EncodeTiled>(p);
}

// `width` x `rows` x `count` elements of 16 bits, boxes of 64 x box_rows
static bool make_map(CUtensorMap *map, alphasparse_cuda_type_t type, const void *p, int64_t width, int64_t rows, int64_t ld,
                     int64_t count, int64_t stride, int box_rows) {
    const EncodeTiled f = encode_tiled();
    if (!f) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)rows, (cuuint64_t)count};
    // distances of dimensions of one element are never used, but have to be legal
    const cuuint64_t strides[2] = {(cuuint64_t)(rows > 1 ? ld * 2 : (width * 2 + 15) / 16 * 16), (cuuint64_t)(count > 1 ? stride * 2 : 16)};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const auto encode = [&] {
        return f(map, type == ALPHA_SPARSE_CUDA_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                 const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (encode()) return true;
    // In a thread whose first call this is nothing has made the device's context current yet, which the runtime does by itself
    // and this function of the driver does not.
    int dev = -1;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encode();
}

static bool takes_tma(const void *p, int64_t ld, int64_t rows, int64_t stride, int64_t count) {
    return address(p) % 16 == 0 && (rows <= 1 || ld % 8 == 0) && (count <= 1 || (stride % 8 == 0 && stride < (int64_t)1 << 38));
}

static cudaError_t multiprocessors(int *n) {
    int dev;
    const cudaError_t e = cudaGetDevice(&dev);
    return e != cudaSuccess ? e : cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev);
}

// Fills what follows from the tile, and launches.
template <int FORM, bool PAIR, bool W_K, bool ANY, typename T, typename TO>
static cudaError_t launch_mm(alphasparse_cuda_type_t type, MmShape s, int64_t most_tiles, const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &c,
                             TO *out,
                             int64_t ldo, int64_t stride_o, cudaStream_t st) {
    constexpr bool a_k = FORM == kRows && W_K, b_k = FORM == kRows;
    constexpr int most_smem = 232448 - 12288;  // tables and barriers are in what is left
    const int half = PAIR ? s.n / 2 : s.n;
    s.stage_bytes = (unsigned)(kMmM * kMmK + (b_k ? half : (half + 63) / 64 * 64) * kMmK) * 2;
    s.stages = std::min<int>(kMmMostStages, (most_smem - 1024) / (int)s.stage_bytes);
    const unsigned format = type == ALPHA_SPARSE_CUDA_TYPE_BF16 ? 1 : 0;
    s.instruction = 1u << 4 | format << 7 | format << 10 | (a_k ? 0u : 1u << 15) | (b_k ? 0u : 1u << 16) |
                    (unsigned)((PAIR ? 2 * kMmM : kMmM) >> 4) << 24;
    s.acc_stride = 256;
    s.vectors = address(out) % 16 == 0 && ldo * (int64_t)sizeof(TO) % 16 == 0 && (FORM != kGradient || stride_o * (int64_t)sizeof(TO) % 16 == 0);
    const auto kernel = expert_mm_kernel<FORM, PAIR, W_K, ANY, T, TO>;
    const int smem = 1024 + s.stages * (int)s.stage_bytes;
    int sms = 0;
    cudaError_t e = multiprocessors(&sms);
    // the most that any call takes, the same from every thread: a call with small stages must not lower it under another's launch
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute cluster[1];
    cluster[0].id = cudaLaunchAttributeClusterDimension;
    cluster[0].val.clusterDim.x = 2, cluster[0].val.clusterDim.y = 1, cluster[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(PAIR ? 2 * std::min<int64_t>(sms / 2, most_tiles) : std::min<int64_t>(sms, most_tiles)));
    config.blockDim = dim3(ANY ? kMmThreadsAny : kMmThreads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = st;
    config.attrs = cluster;
    config.numAttrs = PAIR ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, a, b, c, s, out, ldo, stride_o);
}

static int64_t up_to(int64_t v, int64_t unit) { return (v + unit - 1) / unit * unit; }

}  // namespace asb

using namespace asb;

static bool mm_sizes_fit(int64_t experts, int64_t rows, int64_t a, int64_t b) {
    return experts >= 1 && rows >= 0 && rows <= kMostRows && a >= 0 && a <= kMostWidth && b >= 0 && b <= kMostWidth;
}

// the weights of all experts as one operand: rows within an expert are checked here
static alphasparse_status_t check_weights(const char *call, int64_t out, int64_t in, int64_t ld, int64_t stride, int64_t experts) {
    if ((out > 1 && ld < in) || ld > kMostStride || (experts > 1 && stride < (out > 0 ? (out - 1) * ld + in : 0)) || stride >= (int64_t)1 << 40) {
        char msg[160];
        snprintf(msg, sizeof(msg), "%s: leading dimension below the width, or matrices of the experts that overlap", call);
        record_error(msg);
        return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    }
    return ALPHA_SPARSE_STATUS_SUCCESS;
}
static Operand weights_operand(const void *w, int64_t experts, int64_t out, int64_t in, int64_t ld, int64_t stride, size_t elem, bool written) {
    const bool any = experts > 0 && out > 0 && in > 0;
    return Operand{w, any ? 1 : 0, any ? (experts - 1) * stride + (out - 1) * ld + in : 0, 0, elem, written};
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_mm(alphasparse_operation_t operation, alphasparse_cuda_type_t type, int64_t experts,
                                                           int64_t rows, const int32_t *offsets, int64_t out, int64_t in, const void *x,
                                                           int64_t ldx, const void *w, int64_t ldw, int64_t stride_w, void *y, int64_t ldy) {
    const size_t eb = type_bytes(type);
    if (!eb || !mm_sizes_fit(experts, rows, out, in)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (operation != ALPHA_SPARSE_OPERATION_NON_TRANSPOSE && operation != ALPHA_SPARSE_OPERATION_TRANSPOSE) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (experts > kMostExperts) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    const bool trans = operation == ALPHA_SPARSE_OPERATION_TRANSPOSE;
    const int64_t features = trans ? out : in, reduced = trans ? in : out;
    if (rows == 0 || features == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    alphasparse_status_t status = check_weights("alphasparse_cuda_expert_mm", out, in, ldw, stride_w, experts);
    if (status != ALPHA_SPARSE_STATUS_SUCCESS) return status;
    status = check_operands("alphasparse_cuda_expert_mm", {{offsets, 1, experts + 1, experts + 1, sizeof(int), false},
                                                           {x, rows, reduced, ldx, eb, false},
                                                           weights_operand(w, experts, out, in, ldw, stride_w, eb, false),
                                                           {y, rows, features, ldy, eb, true}});
    if (status != ALPHA_SPARSE_STATUS_SUCCESS) return status;
    cudaStream_t st = current_stream();
    cudaError_t e = cudaSuccess;
    if (eb == 2 && reduced > 0) {
        MmShape s{};
        s.offsets = offsets, s.experts = (int)experts, s.rows = rows, s.m_size = (int)features, s.reduced = (int)reduced;
        const bool any = !takes_tma(x, ldx, rows, 0, 1) || !takes_tma(w, ldw, out, stride_w, experts);
        // Many rows an expert: two SMs on a tile.  Few: the weights are what has to be read, by as many SMs as there are; narrow
        // tiles leave room for more of them on their way.  The mean is over all rows of x: how many of them the offsets name is
        // known on the device alone.  (us by tiles of 32 / 64 / 128 / two SMs, L2 flushed before each; 64 experts of 1408 x 2048:
        // 16 rows each 80 / 81 / 81 / 87, 32: 86 / 81 / 83 / 87, 64: 119 / 85 / 85 / 89, 96: 152 / 103 / 91 / 91,
        // 192: 265 / 161 / 114 / 95.  8 experts of 4096 x 4096: 16: 65 / 65 / 67 / 69, 64: 96 / 73 / 69 / 69, 96: 124 / 85 / 69 / 69,
        // 128: 136 / 97 / 81 / 71, 192: 194 / 121 / 91 / 85.  Up to 96 rows 128 and two SMs are within 8 % of one another.)
        const int64_t mean = (rows + experts - 1) / experts;
        const bool pair = mean > 64 && !any;
        s.n = pair ? 256 : mean <= 16 ? 32 : mean <= 32 ? 64 : 128;
        const int m = pair ? 2 * kMmM : kMmM;
        s.m_tiles = (int)((features + m - 1) / m);
        const int64_t row_tiles = rows / s.n + std::min(experts, rows), tiles = row_tiles * s.m_tiles;
        if (tiles > 0x7fffffff - 4096) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
        CUtensorMap mx{}, mx16{}, mw{};
        if (any) {
            s.a = w, s.lda = ldw, s.stride_a = stride_w, s.b = x, s.ldb = ldx;
            s.all_a = window(w, 1, (experts - 1) * stride_w + (out - 1) * ldw + in, 0, eb);
            s.all_b = window(x, rows, reduced, ldx, eb);
        } else if (!make_map(&mx, type, x, reduced, rows, ldx, 1, 0, 64) || !make_map(&mx16, type, x, reduced, rows, ldx, 1, 0, 16) ||
                   !make_map(&mw, type, w, in, out, ldw, experts, stride_w, trans ? kMmM : kMmK)) {
            record_error("alphasparse_cuda_expert_mm: no tensor map");
            return ALPHA_SPARSE_STATUS_EXECUTION_FAILED;
        }
        const auto go = [&](auto t) {
            using T = decltype(t);
            if (any && trans) e = launch_mm<kRows, false, true, true, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
            else if (any) e = launch_mm<kRows, false, false, true, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
            else if (pair && trans) e = launch_mm<kRows, true, true, false, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
            else if (pair) e = launch_mm<kRows, true, false, false, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
            else if (trans) e = launch_mm<kRows, false, true, false, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
            else e = launch_mm<kRows, false, false, false, T, T>(type, s, tiles, mw, mx, mx16, (T *)y, ldy, 0, st);
        };
        if (type == ALPHA_SPARSE_CUDA_TYPE_F16) go(__half());
        else go(__nv_bfloat16());
    } else {
        const int64_t row_tiles = rows / kPlainTile + std::min(experts, rows);
        const dim3 grid((unsigned)((features + kPlainTile - 1) / kPlainTile), (unsigned)std::min<int64_t>(row_tiles, 32768),
                        (unsigned)((row_tiles + 32767) / 32768));
        const auto go = [&](auto t) {
            using T = decltype(t);
            const auto kernel = trans ? expert_mm_plain_kernel<T, T, false, true, true> : expert_mm_plain_kernel<T, T, false, true, false>;
            kernel<<<grid, 256, 0, st>>>(offsets, (int)experts, rows, 0, (int)features, (int)reduced, (const T *)x, ldx, 0, (const T *)w, ldw, stride_w,
                                         0.f, (T *)y, ldy, 0);
            e = cudaGetLastError();
        };
        ASB_BY_TYPE(type, go)
    }
    ASB_CUDA_OR(e, ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    count_launch();
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_mm_grad(alphasparse_cuda_type_t type, alphasparse_cuda_type_t weight_type, int64_t experts,
                                                                int64_t rows, const int32_t *offsets, int64_t out, int64_t in, const void *dy,
                                                                int64_t lddy, const void *x, int64_t ldx, float beta, void *dw, int64_t ldw,
                                                                int64_t stride_w) {
    const size_t eb = type_bytes(type), ob = type_bytes(weight_type);
    if (!eb || !ob || !mm_sizes_fit(experts, rows, out, in)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (experts > kMostExperts || (weight_type != type && weight_type != ALPHA_SPARSE_CUDA_TYPE_F32)) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    if (out == 0 || in == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    alphasparse_status_t status = check_weights("alphasparse_cuda_expert_mm_grad", out, in, ldw, stride_w, experts);
    if (status != ALPHA_SPARSE_STATUS_SUCCESS) return status;
    status = check_operands("alphasparse_cuda_expert_mm_grad", {{offsets, 1, experts + 1, experts + 1, sizeof(int), false},
                                                                {dy, rows, out, lddy, eb, false},
                                                                {x, rows, in, ldx, eb, false},
                                                                weights_operand(dw, experts, out, in, ldw, stride_w, ob, true)});
    if (status != ALPHA_SPARSE_STATUS_SUCCESS) return status;
    cudaStream_t st = current_stream();
    cudaError_t e = cudaSuccess;
    if (eb == 2 && rows > 0) {
        MmShape s{};
        s.offsets = offsets, s.experts = (int)experts, s.rows = rows, s.m_size = (int)in, s.n_size = (int)out, s.beta = beta;
        const bool any = !takes_tma(dy, lddy, rows, 0, 1) || !takes_tma(x, ldx, rows, 0, 1);
        const int64_t m = any ? kMmM : 2 * kMmM, n = any ? 128 : 256;
        s.m_tiles = (int)((in + m - 1) / m);
        s.n_tiles = (int)((out + n - 1) / n);
        s.n = (int)up_to((out + s.n_tiles - 1) / s.n_tiles, any ? 16 : 32);  // equal tiles of the columns of dy
        const int64_t tiles = experts * s.m_tiles * s.n_tiles;
        if (tiles > 0x7fffffff - 4096) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
        CUtensorMap my{}, mx{};
        if (any) {
            s.a = x, s.lda = ldx, s.b = dy, s.ldb = lddy;
            s.all_a = window(x, rows, in, ldx, eb), s.all_b = window(dy, rows, out, lddy, eb);
        } else if (!make_map(&my, type, dy, out, rows, lddy, 1, 0, kMmK) || !make_map(&mx, type, x, in, rows, ldx, 1, 0, kMmK)) {
            record_error("alphasparse_cuda_expert_mm_grad: no tensor map");
            return ALPHA_SPARSE_STATUS_EXECUTION_FAILED;
        }
        const auto go = [&](auto t) {
            using T = decltype(t);
            const auto with_output = [&](auto o) {
                using TO = decltype(o);
                if (any) e = launch_mm<kGradient, false, false, true, T, TO>(type, s, tiles, mx, my, my, (TO *)dw, ldw, stride_w, st);
                else e = launch_mm<kGradient, true, false, false, T, TO>(type, s, tiles, mx, my, my, (TO *)dw, ldw, stride_w, st);
            };
            if (weight_type == ALPHA_SPARSE_CUDA_TYPE_F32) with_output((float)0);
            else with_output(t);
        };
        if (type == ALPHA_SPARSE_CUDA_TYPE_F16) go(__half());
        else go(__nv_bfloat16());
    } else {
        const int64_t tiles = (in + kPlainTile - 1) / kPlainTile * ((out + kPlainTile - 1) / kPlainTile);
        if (tiles > 0x7fffffff) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
        const dim3 grid((unsigned)tiles, 1, (unsigned)experts);
        const auto go = [&](auto t) {
            using T = decltype(t);
            if (weight_type == ALPHA_SPARSE_CUDA_TYPE_F32)
                expert_mm_plain_kernel<T, float, true, false, false><<<grid, 256, 0, st>>>(offsets, (int)experts, rows, (int)out, (int)in, 0, (const T *)dy, lddy, 0,
                                                                                        (const T *)x, ldx, 0, beta, (float *)dw, ldw, stride_w);
            else
                expert_mm_plain_kernel<T, T, true, false, false><<<grid, 256, 0, st>>>(offsets, (int)experts, rows, (int)out, (int)in, 0, (const T *)dy, lddy, 0,
                                                                                    (const T *)x, ldx, 0, beta, (T *)dw, ldw, stride_w);
            e = cudaGetLastError();
        };
        ASB_BY_TYPE(type, go)
    }
    ASB_CUDA_OR(e, ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    count_launch();
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_mm_status(int *status, int clear) {
    if (!status) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;
    cudaStream_t st = current_stream();
    if (being_captured(st)) {  // it waits; and refused here, the capture goes on
        record_error("alphasparse_cuda_expert_mm_status: the library stream is being captured");
        return ALPHA_SPARSE_STATUS_EXECUTION_FAILED;
    }
    static std::mutex one_at_a_time;  // the word for the host is one per device
    std::lock_guard<std::mutex> lock(one_at_a_time);
    void *word = nullptr;
    ASB_CUDA_OR(cudaGetSymbolAddress(&word, g_expert_mm_told), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    tell_status_kernel<<<1, 1, 0, st>>>(clear);
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    count_launch();
    int told = 0;
    ASB_CUDA_OR(cudaMemcpyAsync(&told, word, sizeof(int), cudaMemcpyDeviceToHost, st), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    ASB_CUDA_OR(cudaStreamSynchronize(st), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    *status = told;
    return ALPHA_SPARSE_STATUS_SUCCESS;
}
