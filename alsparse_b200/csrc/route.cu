// Routing of tokens to experts: scores of the logits, choice of the top k, weights, and the gradient of the weights.  The
// outcome is a sparse matrix of k entries per token (index, weight) that expert_plan, dispatch and combine (experts.cu)
// multiply by.  No counterpart in the reference.
//
// The choice is the one that 64-bit arithmetic makes.  Without a bias a score grows with its logit, so logits are compared,
// exactly.  With a bias the keys score + bias are formed in 32 bits first, and a token of which two keys that matter lie
// closer together than 32 bits can tell apart is decided again in 64 (about one token in a hundred of unrelated keys).
#include <algorithm>

#include "rows.h"

namespace asb {

constexpr int kRouteWarps = 4;
constexpr int kSortedItems = 8;  // logits a lane that it sorts; more: the largest one by one (512 experts, 8 of them: sorted 87 us, so 59 us)
constexpr unsigned kAll = 0xffffffffu;

// Keys as unsigned numbers of the same order.  0 stands for an expert that cannot be chosen (a logit or key of minus
// infinity, a group left out, one already chosen); a NaN comes before everything else; the two zeros are one.
__device__ __forceinline__ unsigned order_of(float key) {
    const unsigned b = __float_as_uint(key + 0.f), o = b ^ (unsigned)((int)b >> 31 | 0x80000000);
    return key > -INFINITY ? o : key == -INFINITY ? 0u : 0xffffffffu;
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
    int group_lanes;  // lanes that hold a group, where every group fills a power of two of them; else 0
    bool sigmoid, renorm, packs, bias_packs;
    float scale;
    int space;  // doubles of shared memory a warp
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
    if (m == -INFINITY) m = 0;  // every expert is masked: exp gives zeros
    F s = 0;
#pragma unroll
    for (int i = 0; i < I; i++) s += exp_of((F)x[i] - m);
    *top = m, *sum = warp_sum(s);
}

// Elements in one access of a lane's I logits
template <typename T, int I>
constexpr __host__ __device__ int route_pack() {
    int p = 1;
    while (p * 2 * (int)sizeof(T) <= 16 && I % (p * 2) == 0) p *= 2;
    return p;
}

// Lane l takes the logits of experts l I, ..., l I + I - 1; minus infinity behind the last expert
template <typename T, int I>
__device__ __forceinline__ void load_logits(const T *row, int experts, bool packs, float (&x)[I]) {
    const int first = (threadIdx.x & 31) * I;
    constexpr int P = route_pack<T, I>();
    if (packs && first + I <= experts) {
#pragma unroll
        for (int i = 0; i < I; i += P) {
            float f[P];
            unpack<T, P>(load_pack<T, P>(row + first + i), f);
#pragma unroll
            for (int j = 0; j < P; j++) x[i + j] = f[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < I; i++) x[i] = first + i < experts ? to_float(row[first + i]) : -INFINITY;
    }
}

// The best runs, for lane g < groups: whether run g is among the top_groups, from the values and orders that the lanes of the
// groups read out of shared memory (one padding element per group).  Returns the mask of the runs; *value and *rank: this
// lane's run.
template <typename F, bool BIAS>
__device__ __forceinline__ unsigned best_groups(const RouteShape &sh, const F *s_key, F *value, int *rank) {
    using O = decltype(order_of(F(0)));
    const int lane = threadIdx.x & 31;
    O worth = 0;
    *value = -INFINITY;
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
        // half the sum of two keys, which no finite ones take out of range
        *value = BIAS ? F(.5) * v1 + (second != 0 ? F(.5) * v2 : F(0)) : v1;
        worth = first == 0 ? 0 : order_of(*value);
    }
    int ahead = 0;
    for (int g = 0; g < sh.groups; g++) {
        const O w = __shfl_sync(kAll, worth, g);
        ahead += w > worth || (w == worth && g < lane);
    }
    *rank = lane < sh.groups ? ahead : sh.groups;
    return __ballot_sync(kAll, lane < sh.groups && ahead < sh.top_groups);
}

// Keys of 32 bits are off by a few units in the last place of a score (at most 1; exp and quotient are the fast ones, within
// some eight units of it in all) and of the sum with the bias: two that are further apart than this stand as they do in 64.
__device__ __forceinline__ bool apart(float a, float b) { return a - b > 4e-6f * (1.f + fabsf(b)); }

// The score of a key: in 32 bits by the fast functions, since what they may get wrong is decided again
__device__ __forceinline__ float key_score(const RouteShape &sh, float x, float top, float sum) {
    return sh.sigmoid ? __fdividef(1.f, 1.f + __expf(-x)) : __fdividef(__expf(x - top), sum);
}
__device__ __forceinline__ double key_score(const RouteShape &sh, double x, double top, double sum) {
    return sh.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum;
}

// Experts of one token by keys of type F, in a warp; lane j gets the j-th choice, -1 where nothing is left.  The plain way: the
// largest key that is left, k times.  Returns false when 32-bit keys do not decide it.
template <typename F, int I, bool BIAS>
__device__ __forceinline__ bool choose(const RouteShape &sh, const float (&x)[I], const float *bias, F top, F sum,
                                       F *s_key, int *choice) {
    using O = decltype(order_of(F(0)));
    constexpr bool check = BIAS && sizeof(F) == 4;
    const int lane = threadIdx.x & 31;
    O key[I];
    int group = lane * I / sh.group_size, within = lane * I - group * sh.group_size;
    const int group0 = group, within0 = within;
#pragma unroll
    for (int i = 0; i < I; i++) {
        const int e = lane * I + i;
        F v = (F)x[i];
        if (BIAS && e < sh.experts && x[i] != -INFINITY)
            v = key_score(sh, v, top, sum) + (F)__ldg(bias + e);
        key[i] = e < sh.experts ? order_of(v) : 0;
        // the values themselves go through shared memory to the lanes of the groups
        if (sh.groups > 1 && e < sh.experts) s_key[e + group] = v;
        if (++within == sh.group_size) within = 0, group++;
    }
    if (sh.groups > 1) {
        __syncwarp();
        F value;
        int rank;
        const unsigned mask = best_groups<F, BIAS>(sh, s_key, &value, &rank);
        if (check) {
            // the last group that is in and the first that is not
            const unsigned in = __ballot_sync(kAll, rank == sh.top_groups - 1), out = __ballot_sync(kAll, rank == sh.top_groups);
            const float a = (float)__shfl_sync(kAll, value, __ffs(in) - 1), b = (float)__shfl_sync(kAll, value, __ffs(out) - 1);
            if (!apart(a, b) && b != -INFINITY) return false;
        }
        group = group0, within = within0;
#pragma unroll
        for (int i = 0; i < I; i++) {
            if (!(mask >> (group & 31) & 1u)) key[i] = 0;
            if (++within == sh.group_size) within = 0, group++;
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
            if (j > 0 && w != 0 && !apart(before, v)) return false;
            before = v;
        }
        if (w == 0 || j == sh.k) break;
        int e = 0x7fffffff;
        if (best == w) {
#pragma unroll
            for (int i = I - 1; i >= 0; i--)
                if (key[i] == w) e = lane * I + i;
        }
        e = (int)__reduce_min_sync(kAll, (unsigned)e);
        if (lane == j) *choice = e;
        if (e >= lane * I && e < lane * I + I) {
            best = 0;
#pragma unroll
            for (int i = 0; i < I; i++) {
                if (e == lane * I + i) key[i] = 0;
                best = key[i] > best ? key[i] : best;
            }
        }
    }
    return true;
}

// The same in 64 bits, for the tokens that need it; out of line, so that it costs the others no registers
template <typename T, int I>
__device__ __noinline__ int choose_in_64(const RouteShape &sh, const T *row, const float *bias, double *s_key) {
    float x[I];
    load_logits<T, I>(row, sh.experts, sh.packs, x);
    double top = 0, sum = 1;
    if (!sh.sigmoid) softmax_stats<double, I>(x, &top, &sum);
    int choice;
    choose<double, I, true>(sh, x, bias, top, sum, s_key, &choice);
    return choice;
}

// Sorts the lane's keys, highest first, by a merging network (Batcher's odd-even merge sort; comparisons that reach behind I
// are left out, which sorts any I)
template <int I>
__device__ __forceinline__ void sort_keys(unsigned long long (&key)[I]) {
#pragma unroll
    for (int p = 1; p < I; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < I; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < I && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const unsigned long long a = key[i + j], b = key[i + j + q];
                        key[i + j] = a > b ? a : b;
                        key[i + j + q] = a > b ? b : a;
                    }
}

// 32-bit keys, up to eight a lane: each lane sorts its own (order above, the complement of the index below, so that equal
// keys go by index) and leaves them in shared memory; the highest head is taken k times, its lane reads its next.  Bound by
// instructions.  (256 experts in 8 groups, 8 of them, 32,768 tokens: the plain way 104 us, sorted keys moved up in
// registers 55 us, so 47 us.)
template <int I, bool BIAS>
__device__ __forceinline__ bool choose_sorted(const RouteShape &sh, const float (&x)[I], const float *bias, float top, float sum,
                                              double *s_space, int *choice, float *logit) {
    const int lane = threadIdx.x & 31;
    const float over = 1.f / sum;
    float v[I];
    if (BIAS) {
        load_logits<float, I>(bias, sh.experts, sh.bias_packs, v);  // minus infinity behind the last expert
#pragma unroll
        for (int i = 0; i < I; i++) {
            const float s = (sh.sigmoid ? __fdividef(1.f, 1.f + __expf(-x[i])) : __expf(x[i] - top) * over) + v[i];
            v[i] = x[i] == -INFINITY ? -INFINITY : s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < I; i++) v[i] = x[i];
    }
    unsigned order[I];
#pragma unroll
    for (int i = 0; i < I; i++) order[i] = order_of(v[i]);
    if (sh.groups > 1 && sh.group_lanes == 0) {
        float *s_key = reinterpret_cast<float *>(s_space);
        int group = lane * I / sh.group_size, within = lane * I - group * sh.group_size;
        const int group0 = group, within0 = within;
#pragma unroll
        for (int i = 0; i < I; i++) {
            if (lane * I + i < sh.experts) s_key[lane * I + i + group] = v[i];
            if (++within == sh.group_size) within = 0, group++;
        }
        __syncwarp();
        float value;
        int rank;
        const unsigned mask = best_groups<float, BIAS>(sh, s_key, &value, &rank);
        if (BIAS) {
            const unsigned in = __ballot_sync(kAll, rank == sh.top_groups - 1), out = __ballot_sync(kAll, rank == sh.top_groups);
            const float a = __shfl_sync(kAll, value, __ffs(in) - 1), b = __shfl_sync(kAll, value, __ffs(out) - 1);
            if (!apart(a, b) && b != -INFINITY) return false;
        }
        group = group0, within = within0;
#pragma unroll
        for (int i = 0; i < I; i++) {
            if (!(mask >> (group & 31) & 1u)) order[i] = 0;
            if (++within == sh.group_size) within = 0, group++;
        }
        __syncwarp();
    }
    unsigned long long key[I];
#pragma unroll
    for (int i = 0; i < I; i++) key[i] = (unsigned long long)order[i] << 32 | (0xffffffffu - (unsigned)(lane * I + i));
    sort_keys<I>(key);
    if (sh.groups > 1 && sh.group_lanes != 0) {
        // the two highest of the run, by the lanes that hold it
        unsigned first = (unsigned)(key[0] >> 32), second = I > 1 ? (unsigned)(key[I > 1 ? 1 : 0] >> 32) : 0u;
        for (int o = 1; o < sh.group_lanes; o <<= 1) {
            const unsigned f = __shfl_xor_sync(kAll, first, o), g = __shfl_xor_sync(kAll, second, o);
            second = max(min(first, f), max(second, g));
            first = max(first, f);
        }
        unsigned worth = first;
        if (BIAS) {
            worth = order_of(.5f * key_of(first) + (second != 0 ? .5f * key_of(second) : 0.f));  // halves, as in best_groups
            if (first == 0) worth = 0;
        }
        const int mine = lane / sh.group_lanes;
        int ahead = 0;
        for (int g = 0; g < sh.groups; g++) {
            const unsigned w = __shfl_sync(kAll, worth, g * sh.group_lanes);
            ahead += w > worth || (w == worth && g < mine);
        }
        const bool there = mine < sh.groups, kept = there && ahead < sh.top_groups;
        if (BIAS) {
            const unsigned last = __reduce_min_sync(kAll, kept ? worth : 0xffffffffu), next = __reduce_max_sync(kAll, there && !kept ? worth : 0u);
            if (next != 0 && !apart(key_of(last), key_of(next))) return false;
        }
        if (!kept) key[0] = 0;  // never taken, so none behind it is either
    }
    unsigned long long *mine = reinterpret_cast<unsigned long long *>(s_space) + lane;
#pragma unroll
    for (int i = 1; i < I; i++) mine[32 * i] = key[i];
    unsigned long long head = key[0];
    int next = 1;
    unsigned taken = 0, at = 0, last = 0;
    for (int j = 0; j < sh.k + (BIAS ? 1 : 0); j++) {
        const unsigned w = __reduce_max_sync(kAll, (unsigned)(head >> 32));
        if (w == 0) break;
        if (BIAS && j == sh.k) {
            last = w;
            break;
        }
        const int from = __ffs(__ballot_sync(kAll, (unsigned)(head >> 32) == w)) - 1;  // equal keys: the lowest lane has the lowest index
        const unsigned e = __shfl_sync(kAll, (unsigned)head, from);
        if (lane == j) taken = w, at = e;
        if (lane == from) {
            head = next < I ? mine[32 * next] : 0ull;
            next++;
        }
    }
    if (BIAS) {
        // each choice against the one behind it, the last against the best that was left out
        const unsigned other = __shfl_down_sync(kAll, taken, 1), behind = lane == sh.k - 1 ? last : other;
        if (__any_sync(kAll, taken != 0 && behind != 0 && !apart(key_of(taken), key_of(behind)))) return false;
    }
    *choice = taken != 0 ? (int)(0xffffffffu - at) : -1;
    if (!BIAS) *logit = key_of(taken);
    return true;
}

// Lane j's weight from the logit v of its choice (live: the slot is filled).  Renormalised weights are formed from the
// chosen logits alone, shifted so that the largest term is between 1/2 and 1: no score underflows to 0 / 0.
__device__ __forceinline__ float weight_of(const RouteShape &sh, float v, bool live, float top, float sum) {
    float s;
    if (sh.renorm) {
        const float m = key_of(__reduce_max_sync(kAll, live ? order_of(v) : 0u));  // a NaN leads the order
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

// A warp per token.  (Four tokens a warp one after the other, their weights formed together and the next token's logits
// requested ahead, was no faster: fewer warps to hide the chain of dependent steps of each.)
template <typename T, int I, bool BIAS>
__global__ void __launch_bounds__(kRouteWarps * 32, I <= 8 ? 8 : I <= 16 ? 6 : 1)
    route_kernel(RouteShape sh, int tokens, const T *__restrict__ logits, int64_t ldl, const float *__restrict__ bias,
                 int *__restrict__ index, int64_t ldi, float *__restrict__ weight, int64_t ldw) {
    extern __shared__ double s_space[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + w;
    if (t >= tokens) return;
    double *s_key = s_space + (size_t)w * sh.space;
    const T *row = logits + t * ldl;
    float x[I];
    load_logits<T, I>(row, sh.experts, sh.packs, x);
    float top = 0.f, sum = 1.f;
    if (!sh.sigmoid && (BIAS || !sh.renorm)) softmax_stats<float, I>(x, &top, &sum);
    int choice = -1;
    float v = 0.f;  // the logit of the choice
    bool decided;
    if constexpr (I <= kSortedItems) decided = choose_sorted<I, BIAS>(sh, x, bias, top, sum, s_key, &choice, &v);
    else decided = choose<float, I, BIAS>(sh, x, bias, top, sum, reinterpret_cast<float *>(s_key), &choice);
    if constexpr (BIAS) {
        if (!decided) {
            __syncwarp();
            choice = choose_in_64<T, I>(sh, row, bias, s_key);
        }
    }
    const bool live = choice >= 0;
    if ((BIAS || I > kSortedItems) && live) v = to_float(row[choice]);
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
    const int each = (experts + 31) / 32;
    switch (each) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
        case 8: return f(std::integral_constant<int, 8>{});
    }
    if (each <= 12) f(std::integral_constant<int, 12>{});
    else if (each <= 16) f(std::integral_constant<int, 16>{});
    else if (each <= 24) f(std::integral_constant<int, 24>{});
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
    RouteShape sh{(int)experts, (int)k, limited ? (int)groups : 1, (int)top_groups, (int)(experts / groups), 0,
                  score == ALPHA_SPARSE_CUDA_SCORE_SIGMOID, renormalize != 0, false, address(bias) % 16 == 0, scale, 0};
    cudaStream_t st = current_stream();
    const unsigned blocks = (unsigned)((tokens + kRouteWarps - 1) / kRouteWarps);
    const auto run = [&](auto t) {
        using T = decltype(t);
        with_items(sh.experts, [&](auto items) {
            constexpr int I = decltype(items)::value;
            constexpr uint64_t pack = route_pack<T, I>() * sizeof(T);
            sh.packs = address(logits) % pack == 0 && (uint64_t)ldl * sizeof(T) % pack == 0;
            const int across = sh.group_size / I;
            sh.group_lanes = sh.group_size % I == 0 && (across & (across - 1)) == 0 ? across : 0;
            sh.space = std::max(limited ? sh.experts + sh.groups : 0, I <= kSortedItems ? 32 * I : 0);
            const size_t smem = sizeof(double) * kRouteWarps * (size_t)sh.space;
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
    const RouteShape sh{(int)experts, (int)k, 1, 1, (int)experts, 0, score == ALPHA_SPARSE_CUDA_SCORE_SIGMOID, renormalize != 0, false, false, scale, 0};
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
