// Embedding lookup and the gradient of its table: Y = scale S E and dE = alpha S^T dY + beta dE, S the one-hot matrix of
// the tokens.  S is never stored: the lookup reads the tokens, the gradient sorts their positions by token (the transpose
// of S in CSR form, made for one product) and sums the rows of dY run by run.  No counterpart in the reference.
#include <limits.h>
#include <stdio.h>

#include <algorithm>

#include "rows.h"

namespace asb {

// ---- checks shared by the operators on rows ----------------------------------------------------

// true when `p` is memory the kernels of device `dev` can use: allocated on that device, or managed
static bool memory_of(const void *p, int dev) {
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return false;
    }
    if (at.type == cudaMemoryTypeManaged) return true;
    return at.type == cudaMemoryTypeDevice && at.device == dev;
}

// Whether two operands share memory: their extents meet, and they are not different columns of rows of one length
static bool meet(const Operand &a, const Operand &b) {
    if (a.begin() >= b.end() || b.begin() >= a.end()) return false;
    const uint64_t pitch = (uint64_t)a.ld * a.elem;
    if (pitch == 0 || pitch != (uint64_t)b.ld * b.elem) return true;
    const uint64_t wa = (uint64_t)a.width * a.elem, wb = (uint64_t)b.width * b.elem;
    const uint64_t from = b.begin() >= a.begin() ? (b.begin() - a.begin()) % pitch : (pitch - (a.begin() - b.begin()) % pitch) % pitch;
    return from < wa || from + wb > pitch;
}

alphasparse_status_t check_operands(const char *call, std::initializer_list<Operand> operands) {
    char msg[200];
    for (const Operand &o : operands) {
        if (o.empty()) continue;
        if (!o.p) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;
        if (o.ld > kMostStride || (o.rows > 1 && o.ld < o.width) || o.begin() % o.elem) {
            snprintf(msg, sizeof(msg), "%s: a leading dimension below the width or above 2^31 - 1, or an address that is no multiple of the element's size", call);
            record_error(msg);
            return ALPHA_SPARSE_STATUS_INVALID_VALUE;
        }
    }
    for (const Operand *a = operands.begin(); a != operands.end(); a++)
        for (const Operand *b = operands.begin(); b != a; b++)
            if ((a->written || b->written) && !a->empty() && !b->empty() && meet(*a, *b)) {
                snprintf(msg, sizeof(msg), "%s: an output lies in the place of another operand", call);
                record_error(msg);
                return ALPHA_SPARSE_STATUS_INVALID_VALUE;
            }
    int dev = -1;
    ASB_CUDA_OR(cudaGetDevice(&dev), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    for (const Operand &o : operands)
        if (!o.empty() && !memory_of(o.p, dev)) {
            snprintf(msg, sizeof(msg), "%s takes pointers to memory of the current device only", call);
            record_error(msg);
            return ALPHA_SPARSE_STATUS_INVALID_POINTER;
        }
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

// ---- lookup --------------------------------------------------------------------------------------

// ANY: rows that begin on no 16-byte boundary.  A row of y is cut at the boundaries of its memory and read at whatever shift the
// table's row has to it.  (16,000 rows of 3283 fp16: 2 bytes an access, 16 of
// them in flight, 79 us; four vectors a thread 41 us, two 39 us, one 47 us.)
template <typename T, typename I, int U, bool ANY>
__global__ void __launch_bounds__(kRowThreads)
    embedding_kernel(int rows, const I *__restrict__ token, int64_t inctoken, int64_t vocab, int width, float scale,
                     const T *__restrict__ table, int64_t ldt, Window all, T *__restrict__ y, int64_t ldy, int log) {
    constexpr int E = 16 / sizeof(T);
    const int64_t r = (int64_t)blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log);
    if (r >= rows) return;
    const int64_t t = (int64_t)token[r * inctoken];
    const bool inside = t >= 0 && t < vocab;
    const T *src = table + (inside ? t : 0) * ldt;
    T *dst = y + r * ldy;
    const int v0 = (int)(blockIdx.y * (U << log) + (threadIdx.x & ((1 << log) - 1)));
    const Cut<T> cut(dst, width);
    Pack<T, E> p[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int v = v0 + (u << log);
        p[u] = zero_pack<T, E>();
        if (ANY) {
            if (inside && cut.count(v) > 0) p[u] = load_any<T>(src + cut.begin(v), cut.count(v), all);
        } else if (inside && v * E < width) {
            p[u] = load_pack<T, E>(src + v * E);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int v = v0 + (u << log);
        if (inside && scale != 1.f) {
            float f[E];
            unpack<T, E>(p[u], f);
#pragma unroll
            for (int i = 0; i < E; i++) f[i] *= scale;
            p[u] = pack<T, E>(f);
        }
        if (ANY) {
            store_any<T>(dst + cut.begin(v), cut.count(v), p[u]);
        } else if (v * E < width) {
            store_pack<T, E>(dst + v * E, p[u]);
        }
    }
}

// ---- gradient ------------------------------------------------------------------------------------

constexpr int kGradMostRows = 1024;  // table rows whose tokens one block of the sort collects, at most
constexpr int kGradSortWarps = 32;
constexpr int kGradAhead = 16;       // tokens a lane of the sort requests at a time
constexpr int kGradGroups = 256;     // groups of kGradAhead steps whose steps a warp of the sort remembers
constexpr int kGradPiece = 32;       // sorted positions one block of the sum walks
constexpr int kGradThreads = 128;

// Positions sorted by token, stable, in one launch.  A block owns `own` rows of the table and reads every token: a warp
// takes one contiguous share of them, counts those of each of the block's rows, and after the prefix over warps and rows
// goes through its share again and writes the positions to where they belong.  Tokens below the block's rows are
// counted on the way, so that no block waits for another.  Bound by the latency of a few dependent steps up to some
// 16,384 tokens, whose shares stay in registers between the two passes; beyond, by instructions (51 per step of 32 tokens: 35 us
// for 65,536 tokens, 61 for 131,072), where the second pass leaves out the steps without a token of the block's rows, four of five
// with 148 blocks (the call with 131,072 tokens 114 -> 97 us).
template <typename I>
__global__ void __launch_bounds__(kGradSortWarps * 32)
    tokens_by_row_kernel(int tokens, const I *__restrict__ token, int64_t inctoken, int vocab, int own, int *__restrict__ ptr,
                         int *__restrict__ pos, int *__restrict__ row, int *__restrict__ joins) {
    extern __shared__ int s_count[];  // [warp][row]
    __shared__ int s_sum[kGradSortWarps], s_below[kGradSortWarps];
    __shared__ unsigned short s_hits[kGradSortWarps][kGradGroups];
    let_next_begin();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int base = blockIdx.x * own;
    const int mine = min(own, vocab - base);
    if (blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;  // the list of the sum begins empty
    const int share = (int)(((int64_t)tokens + kGradSortWarps * 32 - 1) / (kGradSortWarps * 32)) * 32;
    const int begin = (int)min((int64_t)tokens, (int64_t)w * share), end = (int)min((int64_t)tokens, (int64_t)begin + share);
    int *count = s_count + w * own;
    int below = 0;
    // 16 steps' tokens of this lane, of those steps that `steps` names; what cannot be a row of the table is the highest number
    unsigned t[kGradAhead];
    const auto request = [&](int i0, unsigned steps) {
        I v[kGradAhead];
        const I *p = token + (i0 + lane) * inctoken;
#pragma unroll
        for (int u = 0; u < kGradAhead; u++, p += 32 * inctoken) {
            v[u] = (I)-1;
            if ((steps >> u & 1) && i0 + u * 32 + lane < end) v[u] = *p;
        }
#pragma unroll
        for (int u = 0; u < kGradAhead; u++) {
            if constexpr (sizeof(I) == 8) t[u] = (unsigned long long)v[u] >> 32 ? ~0u : (unsigned)v[u];
            else t[u] = (unsigned)v[u];
        }
    };
    request(begin, ~0u);
    for (int i = threadIdx.x; i < kGradSortWarps * own; i += blockDim.x) s_count[i] = 0;
    __syncthreads();
    unsigned hits = 0;  // the steps of the last group that hold a token of the block's rows
    int group = 0;
    for (int i0 = begin; i0 < end; i0 += kGradAhead * 32, group++) {
        if (i0 != begin) request(i0, ~0u);
        hits = 0;
#pragma unroll
        for (int u = 0; u < kGradAhead; u++) {
            below += t[u] < (unsigned)base;
            const bool in = t[u] - (unsigned)base < (unsigned)mine;
            if (!__any_sync(0xffffffffu, in)) continue;
            hits |= 1u << u;
            if (in) atomicAdd(&count[t[u] - base], 1);
        }
        if (lane == 0 && group < kGradGroups) s_hits[w][group] = (unsigned short)hits;
    }
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) s_below[w] = below;
    __syncthreads();
    int start = 0;
#pragma unroll
    for (int v = 0; v < kGradSortWarps; v++) start += s_below[v];
    int total = 0;
    if ((int)threadIdx.x < own) {
#pragma unroll 8
        for (int v = 0; v < kGradSortWarps; v++) {
            const int c = s_count[v * own + threadIdx.x];
            s_count[v * own + threadIdx.x] = total;
            total += c;
        }
    }
    int inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
    }
    if (lane == 31) s_sum[w] = inc;
    __syncthreads();
    for (int v = 0; v < w; v++) start += s_sum[v];
    start += inc - total;
    if ((int)threadIdx.x < own) {
#pragma unroll 8
        for (int v = 0; v < kGradSortWarps; v++) s_count[v * own + threadIdx.x] += start;
        if ((int)threadIdx.x < mine) ptr[base + threadIdx.x] = start;
        if (base + (int)threadIdx.x == vocab - 1) ptr[vocab] = start + total;
    }
    __syncthreads();
    group = 0;
    for (int i0 = begin; i0 < end; i0 += kGradAhead * 32, group++) {
        if (share > kGradAhead * 32) {
            hits = group < kGradGroups ? s_hits[w][group] : ~0u;
            request(i0, hits);
        }
#pragma unroll
        for (int u = 0; u < kGradAhead; u++) {
            if (!(hits >> u & 1)) continue;
            const int r = (int)(t[u] - base);
            const bool in = t[u] - (unsigned)base < (unsigned)mine;
            const unsigned same = __match_any_sync(0xffffffffu, in ? r : -1);
            const int lower = __popc(same & ((1u << lane) - 1u));
            const int at = in ? count[r] + lower : 0;
            __syncwarp();
            if (in) {
                pos[at] = i0 + u * 32 + lane;
                row[at] = (int)t[u];
                if (lower == 0) count[r] += __popc(same);
            }
            __syncwarp();
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void finish_row(T *p, const float (&acc)[N], float alpha, float beta) {
    float f[N];
    if (beta != 0.f) unpack<T, N>(load_pack<T, N, true>(p), f);
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = beta != 0.f ? fmaf(alpha, acc[i], beta * f[i]) : alpha * acc[i];
    store_pack<T, N>(p, pack<T, N>(f));
}

// A run of one token that goes over from piece to piece: block `piece` begins it, `pieces` behind go on.  The columns from
// `column` up to `end`: at most kJoinWarps tiles of 128, a warp each, for few pieces; one tile, shared by the warps, for many.
struct Join {
    int row, piece, pieces, column, end;
};
constexpr int kJoinWarps = 8;
constexpr int kJoinFew = 8;
constexpr int kJoinTile = 128;

// Block (piece, column tile): walks kGradPiece sorted positions, several rows of dY requested at a time (and the old values of
// table rows that end among them), and adds up runs of one token in 32 bits, in the order of the tokens.  A run that
// begins and ends in the piece is finished here; what the piece holds of others goes to the partial sums (first slot: of the run
// that came in, second: of the one that goes on), and the run to the list of the join.  The list's order is not fixed, the
// order of every sum is.  The blocks behind take the table's rows that no token names: zeros for beta = 0, beta times
// what is there else.
template <typename T, typename TO, int N, bool BETA>
__global__ void __launch_bounds__(kGradThreads)
    embedding_grad_kernel(int pieces, int tiles, int nv, int vocab, const int *ptr, const int *pos, const int *row,
                          const T *__restrict__ dy, int64_t lddy, float alpha, float beta, TO *__restrict__ dtable, int64_t ldt,
                          float *partial, int64_t ldp, int *joins, Join *join) {
    after_previous();
    let_next_begin();
    const int64_t sums = (int64_t)pieces * tiles;
    if (blockIdx.x >= sums) {
        const int first = (int)(blockIdx.x - sums) * 8;
        const float zero[N] = {};
        for (int r = first; r < min(vocab, first + 8); r++) {
            if (ptr[r] != ptr[r + 1]) continue;
            for (int v = threadIdx.x; v < nv; v += kGradThreads) finish_row<TO, N>(dtable + (int64_t)r * ldt + (int64_t)v * N, zero, 0.f, beta);
        }
        return;
    }
    __shared__ int s_pos[kGradPiece], s_row[kGradPiece + 2];
    const int piece = blockIdx.x / tiles, tile = blockIdx.x - piece * tiles;
    const int count = ptr[vocab], begin = piece * kGradPiece, n = min(kGradPiece, count - begin);
    if (n <= 0) return;
    const int lane = threadIdx.x;
    if (lane < kGradPiece + 2) {
        const int i = begin + lane - 1;
        s_row[lane] = i >= 0 && i < count ? row[i] : -1;
        if (lane < n) s_pos[lane] = pos[begin + lane];
    }
    __syncthreads();
    if (lane == 0 && s_row[n] == s_row[n + 1]) {
        const int r = s_row[n];
        if (ptr[r] >= begin) {  // the run begins here
            const int behind = (ptr[r + 1] - 1) / kGradPiece - piece, width = nv * N;
            const int step = behind <= kJoinFew ? kJoinTile * kJoinWarps : kJoinTile;
            const int c0 = tile * kGradThreads * N, c1 = min(width, c0 + kGradThreads * N);
            int at = atomicAdd(joins, (c1 - c0 + step - 1) / step);
            for (int c = c0; c < c1; c += step) join[at++] = Join{r, piece, behind, c, min(c + step, c1)};
        }
    }
    const int v = tile * kGradThreads + lane;
    if (v >= nv) return;
    const T *src = dy + (int64_t)v * N;
    TO *dst = dtable + (int64_t)v * N;
    float acc[N] = {};
    bool came_in = s_row[0] == s_row[1];
    constexpr int kAhead = BETA ? 4 : 8;
    for (int i0 = 0; i0 < n; i0 += kAhead) {
        Pack<T, N> p[kAhead];
        Pack<TO, N> old[BETA ? kAhead : 1];
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (i0 + u < n) p[u] = load_pack<T, N>(src + s_pos[i0 + u] * lddy);
        if (BETA) {
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                if (i0 + u < n && s_row[i0 + u + 1] != s_row[i0 + u + 2]) old[u] = load_pack<TO, N, true>(dst + (int64_t)s_row[i0 + u + 1] * ldt);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int i = i0 + u;
            if (i >= n) break;
            float f[N];
            unpack<T, N>(p[u], f);
#pragma unroll
            for (int k = 0; k < N; k++) acc[k] += f[k];
            const bool ends = s_row[i + 1] != s_row[i + 2];
            if (!ends && i + 1 < n) continue;
            if (ends && !came_in) {
                if (BETA) unpack<TO, N>(old[BETA ? u : 0], f);
#pragma unroll
                for (int k = 0; k < N; k++) f[k] = BETA ? fmaf(alpha, acc[k], beta * f[k]) : alpha * acc[k];
                store_pack<TO, N>(dst + (int64_t)s_row[i + 1] * ldt, pack<TO, N>(f));
            } else {
                float *to = partial + ((int64_t)piece * 2 + (came_in ? 0 : 1)) * ldp + (int64_t)v * N;
#pragma unroll
                for (int k = 0; k < N; k++) to[k] = acc[k];
            }
            came_in = false;
#pragma unroll
            for (int k = 0; k < N; k++) acc[k] = 0.f;
        }
    }
}

// Runs that cross pieces, one entry of the list at a time: the partial sums of the run, few by one warp, many in equal shares by
// all, whose sums are added in their order.
template <typename TO>
__global__ void __launch_bounds__(kJoinWarps * 32)
    embedding_grad_join_kernel(float alpha, float beta, TO *__restrict__ dtable, int64_t ldt,
                               const float *partial, int64_t ldp, const int *joins, const Join *join) {
    __shared__ float4 s_sum[kJoinWarps][32];
    after_previous();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, count = *joins;
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        const Join j = join[i];
        const bool few = j.pieces <= kJoinFew;
        const int share = few ? j.pieces : (j.pieces + kJoinWarps - 1) / kJoinWarps;
        const int begin = few ? 0 : min(j.pieces, w * share), end = min(j.pieces, begin + share);
        const int c0 = j.column + (few ? w * kJoinTile : 0), c = c0 + lane * 4;
        const float *from = partial + c;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < j.end) {
            if (few || w == 0) acc = *reinterpret_cast<const float4 *>(from + ((int64_t)j.piece * 2 + 1) * ldp);
#pragma unroll 8
            for (int p = begin; p < end; p++) {
                const float4 v = *reinterpret_cast<const float4 *>(from + (int64_t)(j.piece + 1 + p) * 2 * ldp);
                acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
        }
        TO *dst = dtable + (int64_t)j.row * ldt;
        s_sum[w][lane] = acc;
        if (few) __syncwarp();
        else __syncthreads();
        if (few || w == 0) {
#pragma unroll
            for (int q = 0; q < 4; q++) {  // neighbouring lanes, neighbouring columns
                const int at = q * 32 + lane;
                float sum[1] = {0.f};
                if (few) sum[0] = reinterpret_cast<const float *>(s_sum[w])[at];
                else
                    for (int v = 0; v < kJoinWarps; v++) sum[0] += reinterpret_cast<const float *>(s_sum[v])[at];
                if (c0 + at < j.end) finish_row<TO, 1>(dst + c0 + at, sum, alpha, beta);
            }
        }
        __syncthreads();
    }
}

// The pieces of the workspace, each on a 256-byte boundary
struct GradSpace {
    size_t ptr, pos, row, joins, join, partial, bytes;
    int64_t pieces, ldp;
    GradSpace(int64_t tokens, int64_t vocab, int64_t width) {
        const auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
        pieces = (tokens + kGradPiece - 1) / kGradPiece;
        ldp = (width + 3) & ~(int64_t)3;
        ptr = 0;
        pos = up(sizeof(int) * ((size_t)vocab + 1));
        row = pos + up(sizeof(int) * (size_t)tokens);
        joins = row + up(sizeof(int) * (size_t)tokens);
        join = joins + up(sizeof(int));
        // one entry per piece and tile of 128 columns at most
        partial = join + up(sizeof(Join) * (size_t)pieces * (size_t)((width + kJoinTile - 1) / kJoinTile));
        bytes = partial + up(sizeof(float) * 2 * (size_t)pieces * (size_t)ldp);
    }
};

static bool grad_sizes_fit(int64_t tokens, int64_t vocab, int64_t width) {
    return tokens >= 0 && tokens <= kMostRows && vocab >= 0 && vocab <= kMostRows && width >= 0 && width <= kMostWidth;
}

template <typename T, typename TO>
static cudaError_t launch_grad_sums(const GradSpace &sp, char *buffer, int64_t tokens, int64_t vocab, int64_t width, float alpha,
                                    const T *dy, int64_t lddy, float beta, TO *dtable, int64_t ldt, cudaStream_t st) {
    int *ptr = reinterpret_cast<int *>(buffer + sp.ptr), *pos = reinterpret_cast<int *>(buffer + sp.pos),
        *row = reinterpret_cast<int *>(buffer + sp.row), *joins = reinterpret_cast<int *>(buffer + sp.joins);
    Join *join = reinterpret_cast<Join *>(buffer + sp.join);
    float *partial = reinterpret_cast<float *>(buffer + sp.partial);
    const int vb = vector_bytes(sizeof(T), {address(dy), (uint64_t)lddy * sizeof(T), (uint64_t)width * sizeof(T)});
    const int vo = vector_bytes(sizeof(TO), {address(dtable), (uint64_t)ldt * sizeof(TO), (uint64_t)width * sizeof(TO)});
    const auto go = [&](auto n) {
        constexpr int N = decltype(n)::value;
        const int nv = (int)(width / N), tiles = (nv + kGradThreads - 1) / kGradThreads;
        const int64_t blocks = sp.pieces * tiles + (beta == 1.f ? 0 : (vocab + 7) / 8);
        if (blocks <= 0) return cudaSuccess;
        if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
        const auto kernel = beta != 0.f ? embedding_grad_kernel<T, TO, N, true> : embedding_grad_kernel<T, TO, N, false>;
        return launch_behind(kernel, dim3((unsigned)blocks), kGradThreads, 0, st, (int)sp.pieces, tiles, nv, (int)vocab, ptr, pos, row, dy, lddy,
                             alpha, beta, dtable, ldt, partial, sp.ldp, joins, join);
    };
    cudaError_t e;
    constexpr int full = 16 / sizeof(T);
    // A pack of the input becomes one of as many elements of the output: both have to allow it.  Rows on no 16-byte boundary go by
    // one or two elements (16,384 x 2047 bf16 into 65,536 rows of fp32 198 us, 2048 wide 117; beta = 1: 79 and 53).
    if (vb == 16 && vo == 16) e = go(std::integral_constant<int, full>{});
    else if (sizeof(T) == 2 && vb >= 4 && vo >= 2 * (int)sizeof(TO)) e = go(std::integral_constant<int, 2>{});
    else e = go(std::integral_constant<int, 1>{});
    if (e != cudaSuccess) return e;
    count_launch();
    if (sp.pieces > 1) {
        const int64_t most = (sp.pieces - 1) * ((width + kJoinTile - 1) / kJoinTile);
        e = launch_behind(embedding_grad_join_kernel<TO>, dim3((unsigned)std::min<int64_t>(148 * 4, most)), kJoinWarps * 32, 0, st, alpha, beta,
                          dtable, ldt, partial, sp.ldp, joins, join);
        if (e != cudaSuccess) return e;
        count_launch();
    }
    return cudaGetLastError();
}

}  // namespace asb

using namespace asb;

extern "C" alphasparse_status_t alphasparse_cuda_embedding(alphasparse_cuda_index_t index_type, alphasparse_cuda_type_t type,
                                                           int64_t tokens, const void *token, int64_t inctoken, int64_t vocab,
                                                           int64_t width, float scale, const void *table, int64_t ldt, void *y,
                                                           int64_t ldy) {
    const size_t ib = index_bytes(index_type), eb = type_bytes(type);
    if (!ib || !eb || !grad_sizes_fit(tokens, vocab, width) || inctoken < 1) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (tokens == 0 || width == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    const alphasparse_status_t s = check_operands("alphasparse_cuda_embedding", {{token, tokens, 1, inctoken, ib, false},
                                                                               {table, vocab, width, ldt, eb, false},
                                                                               {y, tokens, width, ldy, eb, true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    const int vb = vector_bytes(eb, {address(table), (uint64_t)ldt * eb, address(y), (uint64_t)ldy * eb, (uint64_t)width * eb});
    const bool any = vb < 16;
    const RowShape shape = row_shape(tokens, any ? most_pieces(width, eb) : width * (int64_t)eb / 16, any ? 2 : 4, width * (int64_t)eb < 1024 ? 3 : 5);
    const Window all = window(table, vocab, width, ldt, eb);
    cudaStream_t st = current_stream();
    const auto run = [&](auto t) {
        using T = decltype(t);
        const auto with_index = [&](auto i) {
            using I = decltype(i);
            const auto kernel = any ? (shape.unroll == 1 ? embedding_kernel<T, I, 1, true> : embedding_kernel<T, I, 2, true>)
                                    : (shape.unroll == 1 ? embedding_kernel<T, I, 1, false> : embedding_kernel<T, I, 4, false>);
            kernel<<<shape.grid, kRowThreads, 0, st>>>((int)tokens, (const I *)token, inctoken, vocab, (int)width, scale, (const T *)table, ldt, all,
                                                     (T *)y, ldy, shape.log);
        };
        if (index_type == ALPHA_SPARSE_CUDA_INDEX_I32) with_index((int32_t)0);
        else with_index((int64_t)0);
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_embedding_grad_buffer_size(int64_t tokens, int64_t vocab, int64_t width,
                                                                           size_t *bytes) {
    if (!bytes) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;
    if (!grad_sizes_fit(tokens, vocab, width)) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    *bytes = GradSpace(tokens, vocab, width).bytes;
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_embedding_grad(alphasparse_cuda_index_t index_type, alphasparse_cuda_type_t type,
                                                                alphasparse_cuda_type_t table_type, int64_t tokens,
                                                                const void *token, int64_t inctoken, int64_t vocab,
                                                                int64_t width, float alpha, const void *dy, int64_t lddy,
                                                                float beta, void *dtable, int64_t ldt, void *buffer,
                                                                size_t buffer_bytes) {
    const size_t ib = index_bytes(index_type), eb = type_bytes(type), ob = type_bytes(table_type);
    if (!ib || !eb || !ob || !grad_sizes_fit(tokens, vocab, width) || inctoken < 1) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (table_type != type && table_type != ALPHA_SPARSE_CUDA_TYPE_F32) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    if (vocab == 0 || width == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    const GradSpace sp(tokens, vocab, width);
    if (buffer && (buffer_bytes < sp.bytes || address(buffer) % 16)) {
        record_error("alphasparse_cuda_embedding_grad: the workspace is smaller than alphasparse_cuda_embedding_grad_buffer_size says, or not on a 16-byte boundary");
        return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    }
    const alphasparse_status_t s = check_operands(
        "alphasparse_cuda_embedding_grad", {{token, tokens, 1, inctoken, ib, false},
                                            {dy, tokens, width, lddy, eb, false},
                                            {dtable, vocab, width, ldt, ob, true},
                                            {buffer, 1, (int64_t)sp.bytes, (int64_t)0, 1, true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    cudaStream_t st = current_stream();
    char *space = static_cast<char *>(buffer);
    int *ptr = reinterpret_cast<int *>(space + sp.ptr), *pos = reinterpret_cast<int *>(space + sp.pos),
        *row = reinterpret_cast<int *>(space + sp.row);
    // as many blocks as there are SMs, while their counts fit shared memory, however few rows that leaves each: the fewer it has,
    // the more steps its second pass leaves out (300 rows, 131,072 tokens: 10 blocks of 32 rows 118 us, 100 of 3 97).  Above
    // 148 * 1024 rows there are more blocks than SMs, whose second wave reads all tokens again (64 wide, beta = 1, 16,384 /
    // 131,072 tokens: 151,552 rows 27 / 95 us, 151,553 rows 31 / 100, 303,105 rows 38 / 130)
    const int own = (int)std::min<int64_t>(kGradMostRows, (vocab + 147) / 148);
    const unsigned blocks = (unsigned)((vocab + own - 1) / own);
    const size_t smem = sizeof(int) * kGradSortWarps * (size_t)own;
    const auto sort = [&](auto i) {
        using I = decltype(i);
        cudaError_t e = cudaFuncSetAttribute(tokens_by_row_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(sizeof(int) * kGradSortWarps * kGradMostRows));
        if (e != cudaSuccess) return e;
        tokens_by_row_kernel<I><<<blocks, kGradSortWarps * 32, smem, st>>>((int)tokens, (const I *)token, inctoken, (int)vocab, own, ptr, pos, row,
                                                                          reinterpret_cast<int *>(space + sp.joins));
        return cudaGetLastError();
    };
    ASB_CUDA_OR(index_type == ALPHA_SPARSE_CUDA_INDEX_I32 ? sort((int32_t)0) : sort((int64_t)0), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    count_launch();
    cudaError_t e = cudaSuccess;
    const auto run = [&](auto t) {
        using T = decltype(t);
        if (table_type == ALPHA_SPARSE_CUDA_TYPE_F32)
            e = launch_grad_sums<T, float>(sp, space, tokens, vocab, width, alpha, (const T *)dy, lddy, beta, (float *)dtable, ldt, st);
        else
            e = launch_grad_sums<T, T>(sp, space, tokens, vocab, width, alpha, (const T *)dy, lddy, beta, (T *)dtable, ldt, st);
    };
    ASB_BY_TYPE(type, run)
    ASB_CUDA_OR(e, ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}
