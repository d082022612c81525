// Routing of tokens to experts: scores of the logits, choice of the top k, weights, and the gradient of the weights.  The
// outcome is a sparse matrix of k entries per token (index, weight) that expert_plan, dispatch and combine (experts.cu)
// multiply by.  No counterpart in the reference.
//
// The choice is the one that 64-bit arithmetic makes.  Without a bias a score grows with its logit, so logits are compared,
// exactly.  With a bias the keys score + bias are formed in 32 bits first, and a token of which two keys that matter lie
// closer together than 32 bits can tell apart is decided again in 64 (about one token in a hundred of unrelated keys).
#include "rows.h"

namespace asb {

constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

// Keys as unsigned numbers of the same order.  0 stands for an expert that cannot be chosen (a logit or key of minus
// infinity, a group left out, one already chosen); a NaN comes before everything else; the two zeros are one.
__device__ __forceinline__ unsigned order_of(float key) {
    if (key == -INFINITY) return 0u;
    if (key != key) return 0xffffffffu;
    const unsigned b = __float_as_uint(key + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double key) {
    if (key == -INFINITY) return 0ull;
    if (key != key) return 0xffffffffffffffffull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(key + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float key_of(unsigned o) {
    return o == 0u ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned warp_max(unsigned v) { return __reduce_max_sync(kAll, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const unsigned hi = (unsigned)(v >> 32), top = __reduce_max_sync(kAll, hi);
    const unsigned lo = __reduce_max_sync(kAll, hi == top ? (unsigned)v : 0u);
    return (unsigned long long)top << 32 | lo;
}
template <typename F> __device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
template <typename F> __device__ __forceinline__ F warp_most(F v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
    return v;
}
__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

struct RouteShape {
    int experts, k, groups, top_groups, group_size;
    bool sigmoid, renorm;
    float scale;
};

// softmax over the experts that are not masked: largest logit and sum of the exponentials; NaN goes through
template <typename F, int I>
__device__ __forceinline__ void softmax_stats(const float (&x)[I], F *top, F *sum) {
    F m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < I; i++) m = fmax(m, (F)x[i]), nan |= x[i] != x[i];
    m = warp_most(m);
    if (__any_sync(kAll, nan)) m = NAN;
    F s = 0;
#pragma unroll
    for (int i = 0; i < I; i++) s += x[i] == -INFINITY ? (F)0 : exp_of((F)x[i] - m);
    *top = m, *sum = warp_sum(s);
}

// Experts of one token by keys of type F, in a warp; lane j gets the j-th choice, -1 where nothing is left.  Lane l holds
// the logits of experts l, l + 32, ...  Returns false when 32-bit keys do not decide it.
template <typename F, int I, bool BIAS>
__device__ __forceinline__ bool choose(const RouteShape &sh, const float (&x)[I], const float *bias, F top, F sum,
                                       F *s_key, int *choice) {
    using O = decltype(order_of(F(0)));
    constexpr bool check = BIAS && sizeof(F) == 4;
    const int lane = threadIdx.x & 31;
    O key[I];
#pragma unroll
    for (int i = 0; i < I; i++) {
        const int e = i * 32 + lane;
        F v = (F)x[i];
        if (BIAS && e < sh.experts && x[i] != -INFINITY)
            v = (sh.sigmoid ? (F)1 / ((F)1 + exp_of(-v)) : exp_of(v - top) / sum) + (F)__ldg(bias + e);
        key[i] = e < sh.experts ? order_of(v) : 0;
        // the values themselves go through shared memory to the lanes of the groups
        if (sh.groups > 1 && e < sh.experts) s_key[e + e / sh.group_size] = v;
    }
    // keys of 32 bits are off by a few units in the last place of a score (at most 1) and of the sum with the bias
    const float near = 4e-6f;
    if (sh.groups > 1) {
        __syncwarp();
        O worth = 0;
        F value = -INFINITY;
        if (lane < sh.groups) {
            O first = 0, second = 0;
            F v1 = -INFINITY, v2 = -INFINITY;
            const F *mine = s_key + lane * (sh.group_size + 1);
            for (int i = 0; i < sh.group_size; i++) {
                const F v = mine[i];
                const O o = order_of(v);
                if (o > first) second = first, v2 = v1, first = o, v1 = v;
                else if (o > second) second = o, v2 = v;
            }
            value = BIAS && second != 0 ? v1 + v2 : v1;
            worth = first == 0 ? 0 : order_of(value);
        }
        int ahead = 0;
        for (int g = 0; g < sh.groups; g++) {
            const O w = __shfl_sync(kAll, worth, g);
            ahead += w > worth || (w == worth && g < lane);
        }
        const bool kept = lane < sh.groups && ahead < sh.top_groups;
        const unsigned mask = __ballot_sync(kAll, kept);
        if (check && sh.top_groups < sh.groups) {
            // the last group that is in and the first that is not
            const unsigned in = __ballot_sync(kAll, lane < sh.groups && ahead == sh.top_groups - 1);
            const unsigned out = __ballot_sync(kAll, lane < sh.groups && ahead == sh.top_groups);
            const float a = (float)__shfl_sync(kAll, value, __ffs(in) - 1), b = (float)__shfl_sync(kAll, value, __ffs(out) - 1);
            if (!(a - b > 2.f * near * (1.f + fabsf(a)) || b == -INFINITY)) return false;
        }
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int e = i * 32 + lane;
            if (e < sh.experts && !(mask >> (e / sh.group_size) & 1u)) key[i] = 0;
        }
        __syncwarp();
    }
    O best = 0;
#pragma unroll
    for (int i = 0; i < I; i++) best = key[i] > best ? key[i] : best;
    *choice = -1;
    float before = INFINITY;
    for (int j = 0; j < sh.k + (check ? 1 : 0); j++) {
        const O w = warp_max(best);
        if (check) {
            const float v = key_of((unsigned)w);
            if (j > 0 && w != 0 && !(before - v > near * (1.f + fabsf(v)))) return false;
            before = v;
        }
        if (w == 0 || j == sh.k) break;
        int e = 0x7fffffff;
        if (best == w) {
#pragma unroll
            for (int i = I - 1; i >= 0; i--)
                if (key[i] == w) e = i * 32 + lane;
        }
        e = (int)__reduce_min_sync(kAll, (unsigned)e);
        if (lane == j) *choice = e;
        if ((e & 31) == lane) {
            best = 0;
#pragma unroll
            for (int i = 0; i < I; i++) {
                if (e == i * 32 + lane) key[i] = 0;
                best = key[i] > best ? key[i] : best;
            }
        }
    }
    return true;
}

// Lane j's weight from the logit v of its choice (live: the slot is filled).  Renormalised weights are formed from the
// chosen logits alone, shifted so that the largest term is between 1/2 and 1: no score underflows to 0 / 0.
__device__ __forceinline__ float weight_of(const RouteShape &sh, float v, bool live, float top, float sum) {
    float s;
    if (sh.renorm) {
        bool nan = live && v != v;
        float m = warp_most(live ? v : -INFINITY);
        if (__any_sync(kAll, nan)) m = NAN;
        if (sh.sigmoid) s = m < 0.f ? expf(v - m) / (1.f + expf(v)) : 1.f / (1.f + expf(-v));
        else s = expf(v - m);
        s = live ? s : 0.f;
        const float total = warp_sum(s);
        s = live ? s / total : 0.f;
    } else {
        s = sh.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - top) / sum;
        s = live ? s : 0.f;
    }
    return s;
}

// A warp per token.
template <typename T, int I, bool BIAS>
__global__ void __launch_bounds__(kRouteWarps * 32)
    route_kernel(RouteShape sh, int tokens, const T *__restrict__ logits, int64_t ldl, const float *__restrict__ bias,
                 int *__restrict__ index, int64_t ldi, float *__restrict__ weight, int64_t ldw) {
    extern __shared__ double s_space[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + w;
    if (t >= tokens) return;
    double *s_key = s_space + (size_t)w * (sh.experts + sh.groups);
    const T *row = logits + t * ldl;
    float x[I];
#pragma unroll
    for (int i = 0; i < I; i++) x[i] = i * 32 + lane < sh.experts ? to_float(row[i * 32 + lane]) : -INFINITY;
    float top = 0.f, sum = 1.f;
    if (!sh.sigmoid && (BIAS || !sh.renorm)) softmax_stats<float, I>(x, &top, &sum);
    int choice;
    if (!choose<float, I, BIAS>(sh, x, bias, top, sum, reinterpret_cast<float *>(s_key), &choice)) {
        __syncwarp();
        double top64 = 0, sum64 = 1;
        if (!sh.sigmoid) softmax_stats<double, I>(x, &top64, &sum64);
        choose<double, I, BIAS>(sh, x, bias, top64, sum64, s_key, &choice);
    }
    const bool live = choice >= 0;
    const float v = live ? to_float(row[choice]) : 0.f;
    const float s = weight_of(sh, v, live, top, sum);
    if (lane < sh.k) {
        index[t * ldi + lane] = choice;
        weight[t * ldw + lane] = s * sh.scale;
    }
}

// Gradient of the weights with respect to the logits.  With score s_i and weight w_i = scale s_i: sigmoid
// dx_i = s_i (1 - s_i) scale dw_i; softmax dx_j = s_j (scale dw_j - sum_i scale dw_i s_i), over all experts.  Renormalised,
// r_i = s_i / sum of the chosen s, and c_i = scale r_i (dw_i - sum_j dw_j r_j): sigmoid dx_i = (1 - s_i) c_i; softmax
// dx_i = c_i (what other experts add to the denominators cancels), so in three of the four cases only the chosen
// experts' gradients are not zero.  A warp per token; the row is put together in shared memory.
template <typename T, int I>
__global__ void __launch_bounds__(kRouteWarps * 32)
    route_grad_kernel(RouteShape sh, int tokens, const T *__restrict__ logits, int64_t ldl, const int *__restrict__ index,
                      int64_t ldi, const float *__restrict__ dweight, int64_t ldw, T *__restrict__ dlogits, int64_t ldd) {
    extern __shared__ double s_space[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + w;
    if (t >= tokens) return;
    float *s_row = reinterpret_cast<float *>(s_space) + (size_t)w * sh.experts;
    const T *row = logits + t * ldl;
    const int e = lane < sh.k ? index[t * ldi + lane] : -1;
    const float v = e >= 0 && e < sh.experts ? to_float(row[e]) : 0.f;
    const bool live = e >= 0 && e < sh.experts && v != -INFINITY;
    const float dw = live ? dweight[t * ldw + lane] : 0.f;
    const bool full = !sh.sigmoid && !sh.renorm;
    float x[I], top = 0.f, sum = 1.f;
    if (full) {
#pragma unroll
        for (int i = 0; i < I; i++) x[i] = i * 32 + lane < sh.experts ? to_float(row[i * 32 + lane]) : -INFINITY;
        softmax_stats<float, I>(x, &top, &sum);
    }
    const float r = weight_of(sh, v, live, top, sum);
    const float inner = warp_sum(live ? r * dw : 0.f);  // sum of weight times gradient, before the scale
    float c;
    if (sh.renorm) {
        c = r * (dw - inner);
        if (sh.sigmoid) c *= 1.f / (1.f + expf(v));
    } else {
        c = sh.sigmoid ? r * (1.f / (1.f + expf(v))) * dw : r * dw;
    }
    c = live ? c * sh.scale : 0.f;
    for (int i = lane; i < sh.experts; i += 32) s_row[i] = 0.f;
    __syncwarp();
    for (int j = 0; j < sh.k; j++) {  // in order, so that an expert that is named twice gets both
        const int ej = __shfl_sync(kAll, live ? e : -1, j);
        const float cj = __shfl_sync(kAll, c, j);
        if (ej >= 0 && (ej & 31) == lane) s_row[ej] += cj;
    }
    T *out = dlogits + t * ldd;
    if (full) {
        const float shared = inner * sh.scale;
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int at = i * 32 + lane;
            if (at < sh.experts) out[at] = from_float<T>(x[i] == -INFINITY ? 0.f : s_row[at] - expf(x[i] - top) / sum * shared);
        }
    } else {
        for (int at = lane; at < sh.experts; at += 32) out[at] = from_float<T>(s_row[at]);
    }
}

// Calls f with the number of logits a lane holds
template <typename F>
static void with_items(int experts, F f) {
    if (experts <= 64) f(std::integral_constant<int, 2>{});
    else if (experts <= 128) f(std::integral_constant<int, 4>{});
    else if (experts <= 256) f(std::integral_constant<int, 8>{});
    else if (experts <= 512) f(std::integral_constant<int, 16>{});
    else f(std::integral_constant<int, 32>{});
}

static alphasparse_status_t route_sizes(alphasparse_cuda_score_t score, size_t elem, int64_t tokens, int64_t experts, int64_t k) {
    if (!elem || ((int)score != ALPHA_SPARSE_CUDA_SCORE_SOFTMAX && (int)score != ALPHA_SPARSE_CUDA_SCORE_SIGMOID))
        return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (tokens < 0 || tokens > kMostRows || experts < 1 || k < 1 || k > experts) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    return experts > kMostExperts || k > kMostTopK ? ALPHA_SPARSE_STATUS_NOT_SUPPORTED : ALPHA_SPARSE_STATUS_SUCCESS;
}

}  // namespace asb

using namespace asb;

extern "C" alphasparse_status_t alphasparse_cuda_route(alphasparse_cuda_score_t score, alphasparse_cuda_type_t type, int64_t tokens,
                                                       int64_t experts, const void *logits, int64_t ldl, const float *bias,
                                                       int64_t groups, int64_t top_groups, int64_t k, int renormalize,
                                                       float scale, int32_t *index, int64_t ldi, float *weight, int64_t ldw) {
    const size_t eb = type_bytes(type);
    alphasparse_status_t s = route_sizes(score, eb, tokens, experts, k);
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    if (groups < 1 || experts % groups || top_groups < 1 || top_groups > groups || k > top_groups * (experts / groups))
        return ALPHA_SPARSE_STATUS_INVALID_VALUE;
    if (groups > 32) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
    if (tokens == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    s = check_operands("alphasparse_cuda_route", {{logits, tokens, experts, ldl, eb, false},
                                                  {bias, bias ? 1 : 0, experts, experts, sizeof(float), false},
                                                  {index, tokens, k, ldi, sizeof(int), true},
                                                  {weight, tokens, k, ldw, sizeof(float), true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    // one group, or all of them: no limit
    const bool limited = top_groups < groups;
    const RouteShape sh{(int)experts, (int)k, limited ? (int)groups : 1, (int)top_groups, (int)(experts / groups),
                        score == ALPHA_SPARSE_CUDA_SCORE_SIGMOID, renormalize != 0, scale};
    cudaStream_t st = current_stream();
    const unsigned blocks = (unsigned)((tokens + kRouteWarps - 1) / kRouteWarps);
    const size_t smem = limited ? sizeof(double) * kRouteWarps * (size_t)(sh.experts + sh.groups) : 0;
    const auto run = [&](auto t) {
        using T = decltype(t);
        with_items(sh.experts, [&](auto items) {
            constexpr int I = decltype(items)::value;
            const auto kernel = bias ? route_kernel<T, I, true> : route_kernel<T, I, false>;
            kernel<<<blocks, kRouteWarps * 32, smem, st>>>(sh, (int)tokens, (const T *)logits, ldl, bias, index, ldi, weight, ldw);
        });
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}

extern "C" alphasparse_status_t alphasparse_cuda_route_grad(alphasparse_cuda_score_t score, alphasparse_cuda_type_t type,
                                                            int64_t tokens, int64_t experts, const void *logits, int64_t ldl,
                                                            int64_t k, const int32_t *index, int64_t ldi, int renormalize,
                                                            float scale, const float *dweight, int64_t ldw, void *dlogits,
                                                            int64_t ldd) {
    const size_t eb = type_bytes(type);
    alphasparse_status_t s = route_sizes(score, eb, tokens, experts, k);
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    if (tokens == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
    s = check_operands("alphasparse_cuda_route_grad", {{logits, tokens, experts, ldl, eb, false},
                                                       {index, tokens, k, ldi, sizeof(int), false},
                                                       {dweight, tokens, k, ldw, sizeof(float), false},
                                                       {dlogits, tokens, experts, ldd, eb, true}});
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    const RouteShape sh{(int)experts, (int)k, 1, 1, (int)experts, score == ALPHA_SPARSE_CUDA_SCORE_SIGMOID, renormalize != 0, scale};
    cudaStream_t st = current_stream();
    const unsigned blocks = (unsigned)((tokens + kRouteWarps - 1) / kRouteWarps);
    const size_t smem = sizeof(float) * kRouteWarps * (size_t)sh.experts;
    const auto run = [&](auto t) {
        using T = decltype(t);
        with_items(sh.experts, [&](auto items) {
            constexpr int I = decltype(items)::value;
            route_grad_kernel<T, I><<<blocks, kRouteWarps * 32, smem, st>>>(sh, (int)tokens, (const T *)logits, ldl, index, ldi,
                                                                           dweight, ldw, (T *)dlogits, ldd);
        });
    };
    ASB_BY_TYPE(type, run)
    count_launch();
    ASB_CUDA_OR(cudaGetLastError(), ALPHA_SPARSE_STATUS_EXECUTION_FAILED);
    return ALPHA_SPARSE_STATUS_SUCCESS;
}
