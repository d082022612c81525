// Rows of tokens to their experts and back: the matrix of k entries per token that routing made, as a permutation (plan),
// applied to the tokens' rows (dispatch), and with its weights to the experts' rows (combine, and the gradients).
// No counterpart in the reference.
//
// The (token, choice) pairs stand in the order of their experts, and of the tokens within an expert; slot[t, j] is the row
// of pair (t, j), -1 for an empty choice.  All that follows goes by slot: a token's row is read once and written to its k
// places, or its k rows are read and written once.  Bound by HBM.
#include <algorithm>

#include "rows.h"

namespace asb {

// ---- plan ----------------------------------------------------------------------------------------

constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / 32;
constexpr int kPlanOne = 4096;     // up to so many pairs in one block
constexpr int kPlanKeys = 2048;    // else pairs a block takes at least
constexpr int kPlanMostBlocks = 256;
constexpr int kPlanAhead = 8;      // pairs a lane requests at a time

// Exclusive prefix over the threads of the block; s_sum: one int per warp
__device__ __forceinline__ int plan_scan(int v, int *s_sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
    }
    if (lane == 31) s_sum[w] = inc;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < w; i++) before += s_sum[i];
    __syncthreads();
    return before + inc - v;
}

// A block takes a contiguous share of the pairs and each of its warps a contiguous share of that, counts the pairs of each
// expert per warp, and (PLACE) after the prefix over experts, blocks and warps goes through them again and places them.  With
// more than one block a first launch writes the blocks' counts for the second to read.  Bound by the latency of its steps: a
// lane's pairs are requested eight at a time and stay in registers between the passes where they are no more.
template <bool PLACE>
__global__ void __launch_bounds__(kPlanThreads)
    plan_kernel(int64_t pairs, int64_t share, int experts, int k, const int *__restrict__ index, int64_t ldi,
                int *counts, int *__restrict__ offsets, int *__restrict__ slot, int64_t lds) {
    extern __shared__ int s_count[];  // [warp][expert]
    __shared__ int s_sum[kPlanWarps];
    __shared__ int s_total[kPlanThreads], s_before[kPlanThreads];
    if (!PLACE) let_next_begin();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t first = blockIdx.x * share, last = min(pairs, first + share);
    const int64_t part = (share / kPlanWarps + 31) / 32 * 32;
    const int64_t begin = min(last, first + w * part), end = w == kPlanWarps - 1 ? last : min(last, begin + part);
    int *count = s_count + w * experts;
    int e[kPlanAhead];
    const auto request = [&](int64_t i0) {
#pragma unroll
        for (int u = 0; u < kPlanAhead; u++) {
            const int64_t i = i0 + u * 32 + lane, t = (int64_t)((unsigned)i / (unsigned)k);
            e[u] = i < end ? index[t * ldi + (i - t * k)] : -1;
        }
#pragma unroll
        for (int u = 0; u < kPlanAhead; u++)
            if (e[u] < 0 || e[u] >= experts) e[u] = -1;
    };
    request(begin);
    for (int i = threadIdx.x; i < kPlanWarps * experts; i += kPlanThreads) s_count[i] = 0;
    __syncthreads();
    for (int64_t i0 = begin; i0 < end; i0 += kPlanAhead * 32) {
        if (i0 != begin) request(i0);
#pragma unroll
        for (int u = 0; u < kPlanAhead; u++)
            if (e[u] >= 0) atomicAdd(&count[e[u]], 1);
    }
    __syncthreads();
    const int blocks = gridDim.x, b = blockIdx.x;
    // threads side by side have neighbouring experts; where experts are few, groups of threads share the blocks' counts
    const int across = min(kPlanThreads, (experts + 31) / 32 * 32), parts = kPlanThreads / across;
    const int my_part = threadIdx.x / across, column = threadIdx.x - my_part * across;
    int carry = 0;
    for (int e0 = 0; e0 < experts; e0 += across) {
        const int x = e0 + column;
        int mine = 0;
        if (my_part == 0 && x < experts) {
#pragma unroll
            for (int v = 0; v < kPlanWarps; v++) {
                const int c = s_count[v * experts + x];
                s_count[v * experts + x] = mine;
                mine += c;
            }
        }
        if (!PLACE) {
            if (my_part == 0 && x < experts) counts[(int64_t)b * experts + x] = mine;
            continue;
        }
        int total = mine, before = 0;
        if (blocks > 1) {
            if (e0 == 0) after_previous();  // the counts, and with them whatever came before the first launch
            total = 0;
            if (my_part < parts && x < experts) {
#pragma unroll 8
                for (int v = my_part; v < blocks; v += parts) {
                    const int c = counts[(int64_t)v * experts + x];
                    before += v < b ? c : 0;
                    total += c;
                }
            }
            s_total[threadIdx.x] = total, s_before[threadIdx.x] = before;
            __syncthreads();
            if (my_part == 0) {
                for (int v = 1; v < parts; v++) total += s_total[v * across + column], before += s_before[v * across + column];
            } else {
                total = 0;
            }
        }
        const int start = carry + plan_scan(total, s_sum);
        if (threadIdx.x == kPlanThreads - 1) s_sum[0] = start + total;
        __syncthreads();
        carry = s_sum[0];
        __syncthreads();
        if (my_part == 0 && x < experts) {
#pragma unroll
            for (int v = 0; v < kPlanWarps; v++) s_count[v * experts + x] += start + before;
            if (b == 0) {
                offsets[x] = start;
                if (x == experts - 1) offsets[experts] = start + total;
            }
        }
    }
    if (!PLACE) return;
    __syncthreads();
    for (int64_t i0 = begin; i0 < end; i0 += kPlanAhead * 32) {
        if (part > kPlanAhead * 32 || i0 != begin) request(i0);
#pragma unroll
        for (int u = 0; u < kPlanAhead; u++) {
            if (i0 + u * 32 >= end) break;
            const int64_t i = i0 + u * 32 + lane;
            const unsigned same = __match_any_sync(0xffffffffu, e[u]);
            const int lower = __popc(same & ((1u << lane) - 1u));
            int at = -1;
            if (e[u] >= 0) at = count[e[u]] + lower;
            __syncwarp();
            if (e[u] >= 0 && lower == 0) count[e[u]] += __popc(same);
            __syncwarp();
            if (i < end) {
                const int64_t t = (int64_t)((unsigned)i / (unsigned)k);
                slot[t * lds + (i - t * k)] = at;
            }
        }
    }
}

struct PlanShape {
    int64_t pairs, share;
    int blocks;
    size_t bytes;
    PlanShape(int64_t tokens, int64_t k, int64_t experts) {
        pairs = tokens * k;
        const int64_t want = pairs <= kPlanOne ? 1 : std::min<int64_t>(kPlanMostBlocks, (pairs + kPlanKeys - 1) / kPlanKeys);
        const int64_t unit = 32 * kPlanWarps;  // whole steps of every warp
        share = ((pairs + want - 1) / want + unit - 1) / unit * unit;
        if (share == 0) share = unit;
        blocks = (int)std::max<int64_t>(1, (pairs + share - 1) / share);
        bytes = blocks > 1 ? sizeof(int) * (size_t)blocks * (size_t)experts : 0;
    }
};

// ---- dispatch --------------------------------------------------------------------------------------

// Threads along a token's row as row_shape lays them out: the row is read once and written to every place of the token.  ANY:
// rows that begin on no 16-byte boundary; each place is cut at the boundaries of its memory, and the row read again at the
// shift that it has to it, out of L1.  (12,001 tokens of 6 rows of 2047 fp16: 90 us.  Groups of a warp against those of a block,
// before the ends of rows were loaded as vectors: 154 and 168 us.  Aligned, 2880 wide bf16: 74 us in groups of a warp, so 70.)
template <typename T, int U, bool ANY>
__global__ void __launch_bounds__(kRowThreads)
    dispatch_kernel(int tokens, int k, int width, const T *__restrict__ x, int64_t ldx, Window all, const int *__restrict__ slot,
                    int64_t lds, int64_t rows, T *__restrict__ xs, int64_t ldxs, int log) {
    constexpr int E = 16 / sizeof(T);
    const int64_t t = (int64_t)blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log);
    if (t >= tokens) return;
    const int v0 = (int)(blockIdx.y * (U << log) + (threadIdx.x & ((1 << log) - 1)));
    const T *src = x + t * ldx;
    Pack<T, E> p[U];
    if (!ANY) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = v0 + (u << log);
            if (v * E < width) p[u] = load_pack<T, E>(src + v * E);
        }
    }
    for (int j = 0; j < k; j++) {
        const int at = __ldg(slot + t * lds + j);
        if (at < 0 || at >= rows) continue;
        T *dst = xs + at * ldxs;
        if (ANY) {
            const Cut<T> cut(dst, width);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + (u << log);
                if (cut.count(v) > 0) p[u] = load_any<T>(src + cut.begin(v), cut.count(v), all);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + (u << log), n = cut.count(v);
                if (n > 0) store_any<T>(dst + cut.begin(v), n, p[u]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + (u << log);
                if (v * E < width) store_pack<T, E>(dst + v * E, p[u]);
            }
        }
    }
}

// ---- combine ---------------------------------------------------------------------------------------

// out[t] = sum over j of weight[t, j] y[slot[t, j]] + beta out[t], in 32 bits in the order of j, rounded once.  Eight rows of y
// are requested at a time, 16 bytes of each by a thread: 128 bytes in flight at 64 registers.  (12,001 tokens of 6 rows of 2048
// fp16: four rows of 64 bytes at 138 registers, one block per SM, 94 us; so 65 us.)  ANY, rows that begin on no 16-byte
// boundary: a row's two vectors are loaded where they are added, and blocks enough to fill the SM wait in turn instead: 32
// registers, eight blocks.  (2047 wide: all rows requested first, with their shifts 127 us; 40 registers 94 us; so 82 us.)
constexpr int kCombineAhead = 8;

template <typename T, bool ANY>
__global__ void __launch_bounds__(kRowThreads, ANY ? 8 : 4)
    combine_kernel(int tokens, int k, int width, const T *__restrict__ y, int64_t ldy, Window all, int64_t rows,
                   const int *__restrict__ slot, int64_t lds, const float *__restrict__ weight, int64_t ldw, float beta,
                   T *__restrict__ out, int64_t ldo, int log) {
    constexpr int E = 16 / sizeof(T), A = ANY ? 2 : kCombineAhead;
    const int64_t t = (int64_t)blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log);
    if (t >= tokens) return;
    const int v = (int)((blockIdx.y << log) + (threadIdx.x & ((1 << log) - 1)));
    T *dst = out + t * ldo;
    const Cut<T> cut(dst, width);
    const int *places = slot + t * lds;
    const int from = ANY ? cut.begin(v) : v * E, n = ANY ? cut.count(v) : E;
    if (ANY ? n <= 0 : from >= width) return;
    float acc[E] = {};
    for (int j0 = 0; j0 < k; j0 += A) {
        Pack<T, E> p[A];
        int at[A];
#pragma unroll
        for (int j = 0; j < A; j++) {
            at[j] = j0 + j < k ? __ldg(places + j0 + j) : -1;
            if (at[j] >= rows) at[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < A; j++)
            if (!ANY && at[j] >= 0) p[j] = load_pack<T, E>(y + at[j] * ldy + from);
#pragma unroll
        for (int j = 0; j < A; j++) {
            if (at[j] < 0) continue;
            const float w = weight ? __ldg(weight + t * ldw + j0 + j) : 1.f;
            float f[E];
            unpack<T, E>(ANY ? load_any<T>(y + at[j] * ldy + from, n, all) : p[j], f);
#pragma unroll
            for (int i = 0; i < E; i++) acc[i] = fmaf(w, f[i], acc[i]);
        }
    }
    dst += from;
    if (beta != 0.f) {
        float f[E];
        if (n == E) {
            unpack<T, E>(load_pack<T, E, true>(dst), f);
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) f[i] = i < n ? to_float(dst[i]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < E; i++) acc[i] = fmaf(beta, f[i], acc[i]);
    }
    store_any<T>(dst, n, pack<T, E>(acc));
}

// dy[slot[t, j]] = weight[t, j] dout[t] and dweight[t, j] = <dout[t], y[slot[t, j]]>.  A group of threads of one block has the
// whole row of a token, so that the inner products end in it: lanes, then warps, in a fixed order.  Eight rows at a time,
// as above; their eight inner products are added up over a warp together, each step halving what a lane holds.  (12,001
// tokens of 6 rows of 2048 fp16: four rows at a time 143 us, so 119 us; two blocks per SM instead of three 151 us.)  Groups
// of two warps or more for wide rows: 6000 tokens of 4100 elements 182 us, 217 in single warps.  ANY: each row of dy is cut at the
// boundaries of its memory, and the rows of dout and y read at the shifts that they have to it.
template <typename T, bool ANY>
__global__ void __launch_bounds__(kRowThreads, 3)
    combine_grad_kernel(int tokens, int k, int width, const T *__restrict__ dout, int64_t ldo, Window all_dout,
                        const T *__restrict__ y, int64_t ldy, Window all_y, int64_t rows, const int *__restrict__ slot, int64_t lds,
                        const float *__restrict__ weight, int64_t ldw, T *__restrict__ dy, int64_t lddy,
                        float *__restrict__ dweight, int64_t lddw, int pieces, int log) {
    __shared__ float s_dot[kRowThreads / 32][kCombineAhead];
    constexpr int E = 16 / sizeof(T);
    const int64_t t = (int64_t)blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log);
    const bool mine = t < tokens;  // a block's threads stay together for the barriers
    const int group = 1 << log, me = threadIdx.x & (group - 1), lane = threadIdx.x & 31;
    const T *d_row = dout + t * ldo;
    for (int j0 = 0; j0 < k; j0 += kCombineAhead) {
        int at[kCombineAhead];
        float dot[kCombineAhead] = {};
#pragma unroll
        for (int j = 0; j < kCombineAhead; j++) {
            at[j] = mine && j0 + j < k ? __ldg(slot + t * lds + j0 + j) : -1;
            if (at[j] >= rows) at[j] = -1;
        }
        for (int v = me; mine && v < pieces; v += group) {
            if (ANY) {
#pragma unroll
                for (int j = 0; j < kCombineAhead; j++) {
                    if (at[j] < 0) continue;
                    T *dst = dy + at[j] * lddy;
                    const Cut<T> cut(dst, width);
                    const int from = cut.begin(v), n = cut.count(v);
                    if (n <= 0) continue;
                    const float w = weight ? __ldg(weight + t * ldw + j0 + j) : 1.f;
                    float f[E], g[E];
                    unpack<T, E>(load_any<T>(d_row + from, n, all_dout), f);
                    unpack<T, E>(load_any<T>(y + at[j] * ldy + from, n, all_y), g);
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        if (i < n) dot[j] = fmaf(f[i], g[i], dot[j]);
                        f[i] *= w;
                    }
                    store_any<T>(dst + from, n, pack<T, E>(f));
                }
            } else {
                const int from = v * E;
                const Pack<T, E> d = load_pack<T, E>(d_row + from);
                Pack<T, E> p[kCombineAhead];
#pragma unroll
                for (int j = 0; j < kCombineAhead; j++)
                    if (at[j] >= 0) p[j] = load_pack<T, E>(y + at[j] * ldy + from);
#pragma unroll
                for (int j = 0; j < kCombineAhead; j++) {
                    if (at[j] < 0) continue;
                    const float w = weight ? __ldg(weight + t * ldw + j0 + j) : 1.f;
                    float f[E], g[E];
                    unpack<T, E>(d, f);
                    unpack<T, E>(p[j], g);
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        dot[j] = fmaf(f[i], g[i], dot[j]);
                        f[i] *= w;
                    }
                    store_pack<T, E>(dy + at[j] * lddy + from, pack<T, E>(f));
                }
            }
        }
        if (group < 32) {
#pragma unroll
            for (int j = 0; j < kCombineAhead; j++)
                for (int o = group >> 1; o; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
            if (me == 0 && mine)
#pragma unroll
                for (int j = 0; j < kCombineAhead; j++)
                    if (j0 + j < k) dweight[t * lddw + j0 + j] = at[j] >= 0 ? dot[j] : 0.f;
            continue;
        }
        float half[4], quarter[2], one;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float other = __shfl_xor_sync(0xffffffffu, lane & 16 ? dot[j] : dot[j + 4], 16);
            half[j] = (lane & 16 ? dot[j + 4] : dot[j]) + other;
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float other = __shfl_xor_sync(0xffffffffu, lane & 8 ? half[j] : half[j + 2], 8);
            quarter[j] = (lane & 8 ? half[j + 2] : half[j]) + other;
        }
        one = (lane & 4 ? quarter[1] : quarter[0]) + __shfl_xor_sync(0xffffffffu, lane & 4 ? quarter[0] : quarter[1], 4);
        one += __shfl_xor_sync(0xffffffffu, one, 2);
        one += __shfl_xor_sync(0xffffffffu, one, 1);
        // lanes 4 i to 4 i + 3 hold the warp's sum of product i
        if ((lane & 3) == 0) s_dot[threadIdx.x >> 5][lane >> 2] = one;
        __syncthreads();
        if (me < kCombineAhead && mine && j0 + me < k) {
            float sum = 0.f;
            for (int i = 0; i < group / 32; i++) sum += s_dot[(threadIdx.x >> 5) + i][me];
            dweight[t * lddw + j0 + me] = sum;  // 0 for an empty slot: nothing was added
        }
        __syncthreads();
    }
}

// sizes that the calls on rows of experts share
static bool rows_fit(int64_t tokens, int64_t k, int64_t width, int64_t rows) {
    return tokens >= 0 && k >= 1 && k <= kMostRows && tokens <= kMostRows && tokens * k <= kMostRows && width >= 0 &&
           width <= kMostWidth && rows >= 0 && rows <= kMostRows;
}

}  // namespace asb

using namespace asb;

extern "C" alphasparse_status_t alphasparse_cuda_expert_plan_buffer_size(int64_t tokens, int64_t k, int64_t experts, size_t *bytes) {
    if (!bytes) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;
    if (!rows_fit(tokens, k, 0, 0) || experts < 1) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (experts > kMostExperts) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    *bytes = PlanShape(tokens, k, experts).bytes;
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_plan(int64_t tokens, int64_t k, int64_t experts, const int32_t *index,
                                                             int64_t ldi, int32_t *offsets, int32_t *slot, int64_t lds,
                                                             void *buffer, size_t buffer_bytes) {
    if (!rows_fit(tokens, k, 0, 0) || experts < 1) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (experts > kMostExperts) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    const PlanShape sh(tokens, k, experts);
    if (sh.bytes && buffer && (buffer_bytes < sh.bytes || address(buffer) % sizeof(int))) {
        record_error("alphasparse_cuda_expert_plan: the workspace is smaller than alphasparse_cuda_expert_plan_buffer_size says, or not on a 4-byte boundary");
        return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    }
    const alphasparse_status_t s = check_operands(
        "alphasparse_cuda_expert_plan", {{index, tokens, k, ldi, sizeof(int), false},
                                         {offsets, 1, experts + 1, experts + 1, sizeof(int), true},
                                         {slot, tokens, k, lds, sizeof(int), true},
                                         {buffer, 1, (int64_t)(sh.bytes / sizeof(int)), 0, sizeof(int), true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    cudaStream_t st = current_stream();
    const size_t smem = sizeof(int) * kPlanWarps * (size_t)experts;
    int *counts = static_cast<int *>(buffer);
    if (sh.blocks > 1) {
        ASB_CUDA_OR(cudaFuncSetAttribute(plan_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(int) * kPlanWarps * kMostExperts)),
                    ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
        plan_kernel<false><<<sh.blocks, kPlanThreads, smem, st>>>(sh.pairs, sh.share, (int)experts, (int)k, index, ldi, counts, nullptr, nullptr, 0);
        count_launch();
    }
    ASB_CUDA_OR(cudaFuncSetAttribute(plan_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(int) * kPlanWarps * kMostExperts)),
                ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    if (sh.blocks > 1)
        ASB_CUDA_OR(launch_behind(plan_kernel<true>, dim3(sh.blocks), kPlanThreads, smem, st, sh.pairs, sh.share, (int)experts, (int)k, index, ldi,
                                  counts, offsets, slot, lds),
                    ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    else
        plan_kernel<true><<<1, kPlanThreads, smem, st>>>(sh.pairs, sh.share, (int)experts, (int)k, index, ldi, counts, offsets, slot, lds);
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_dispatch(alphasparse_cuda_type_t type, int64_t tokens, int64_t k, int64_t width,
                                                                 const void *x, int64_t ldx, const int32_t *slot, int64_t lds,
                                                                 int64_t rows, void *xs, int64_t ldxs) {
    const size_t eb = type_bytes(type);
    if (!eb || !rows_fit(tokens, k, width, rows)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (tokens == 0 || width == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    const alphasparse_status_t s = check_operands("alphasparse_cuda_expert_dispatch", {{x, tokens, width, ldx, eb, false},
                                                                                      {slot, tokens, k, lds, sizeof(int), false},
                                                                                      {xs, rows, width, ldxs, eb, true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    const int vb = vector_bytes(eb, {address(x), (uint64_t)ldx * eb, address(xs), (uint64_t)ldxs * eb, (uint64_t)width * eb});
    const bool any = vb < 16;
    const RowShape shape = row_shape(tokens, any ? most_pieces(width, eb) : width * (int64_t)eb / 16, 4, any ? 5 : 8);
    const Window all = window(x, tokens, width, ldx, eb);
    cudaStream_t st = current_stream();
    const auto run = [&](auto t) {
        using T = decltype(t);
        const auto kernel = any ? (shape.unroll == 1 ? dispatch_kernel<T, 1, true> : dispatch_kernel<T, 4, true>)
                                : (shape.unroll == 1 ? dispatch_kernel<T, 1, false> : dispatch_kernel<T, 4, false>);
        kernel<<<shape.grid, kRowThreads, 0, st>>>((int)tokens, (int)k, (int)width, (const T *)x, ldx, all, slot, lds, rows, (T *)xs, ldxs, shape.log);
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_combine(alphasparse_cuda_type_t type, int64_t tokens, int64_t k, int64_t width,
                                                                int64_t rows, const void *y, int64_t ldy, const int32_t *slot,
                                                                int64_t lds, const float *weight, int64_t ldw, float beta,
                                                                void *out, int64_t ldo) {
    const size_t eb = type_bytes(type);
    if (!eb || !rows_fit(tokens, k, width, rows)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (tokens == 0 || width == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    const alphasparse_status_t s = check_operands("alphasparse_cuda_expert_combine", {{y, rows, width, ldy, eb, false},
                                                                                     {slot, tokens, k, lds, sizeof(int), false},
                                                                                     {weight, weight ? tokens : 0, k, ldw, sizeof(float), false},
                                                                                     {out, tokens, width, ldo, eb, true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    const int vb = vector_bytes(eb, {address(y), (uint64_t)ldy * eb, address(out), (uint64_t)ldo * eb, (uint64_t)width * eb});
    const bool any = vb < 16;
    const RowShape shape = row_shape(tokens, any ? most_pieces(width, eb) : width * (int64_t)eb / 16, 1, width * (int64_t)eb < 1024 ? 3 : 5);
    const Window all = window(y, rows, width, ldy, eb);
    cudaStream_t st = current_stream();
    const auto run = [&](auto t) {
        using T = decltype(t);
        const auto kernel = any ? combine_kernel<T, true> : combine_kernel<T, false>;
        kernel<<<shape.grid, kRowThreads, 0, st>>>((int)tokens, (int)k, (int)width, (const T *)y, ldy, all, rows, slot, lds, weight, ldw, beta, (T *)out, ldo,
                                                 shape.log);
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_expert_combine_grad(alphasparse_cuda_type_t type, int64_t tokens, int64_t k, int64_t width,
                                                                     int64_t rows, const void *dout, int64_t ldo, const void *y,
                                                                     int64_t ldy, const int32_t *slot, int64_t lds,
                                                                     const float *weight, int64_t ldw, void *dy, int64_t lddy,
                                                                     float *dweight, int64_t lddw) {
    const size_t eb = type_bytes(type);
    if (!eb || !rows_fit(tokens, k, width, rows)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (tokens == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    const alphasparse_status_t s = check_operands("alphasparse_cuda_expert_combine_grad",
                                                  {{dout, tokens, width, ldo, eb, false},
                                                   {y, rows, width, ldy, eb, false},
                                                   {slot, tokens, k, lds, sizeof(int), false},
                                                   {weight, weight ? tokens : 0, k, ldw, sizeof(float), false},
                                                   {dy, rows, width, lddy, eb, true},
                                                   {dweight, tokens, k, lddw, sizeof(float), true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    const int vb = vector_bytes(eb, {address(dout), (uint64_t)ldo * eb, address(y), (uint64_t)ldy * eb, address(dy),
                                     (uint64_t)lddy * eb, (uint64_t)width * eb});
    const bool any = vb < 16;
    const int64_t pieces = any ? most_pieces(width, eb) : width * (int64_t)eb / 16;
    const int log = row_group(tokens, pieces, 1, pieces < 128 ? 5 : 6);
    const unsigned blocks = (unsigned)((tokens + (kRowThreads >> log) - 1) / (kRowThreads >> log));
    const Window all_dout = window(dout, tokens, width, ldo, eb), all_y = window(y, rows, width, ldy, eb);
    cudaStream_t st = current_stream();
    const auto run = [&](auto t) {
        using T = decltype(t);
        const auto kernel = any ? combine_grad_kernel<T, true> : combine_grad_kernel<T, false>;
        kernel<<<blocks, kRowThreads, 0, st>>>((int)tokens, (int)k, (int)width, (const T *)dout, ldo, all_dout, (const T *)y, ldy, all_y, rows, slot, lds, weight,
                                             ldw, (T *)dy, lddy, dweight, lddw, (int)pieces, log);
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}
