// The norm of all of a model's gradients together, and the gradients scaled down to a limit of it:
//   n = sqrt(sum of g^2 over all values of all tensors),  y = g * (n <= limit ? 1 : limit / n)
//
// The bound is memory: every value is read for the norm and, before any result can be written, the norm has to be
// whole, so every value is read once more.  Two launches: the first leaves one sum for each block, the second adds them
// up again in each block, in the same order, and writes the results.  It walks backwards, from what was read last, and
// finds some of that in L2 (126 MB, which the results take too): of 109 MB float32 it reads 52 from memory, of 55 MB
// bf16 18.
//
// The tensors' table travels as a kernel argument, so a call copies nothing to the device, may be captured and needs
// no table that lives on.  Tensors differ in length from one value to millions; laid end to end, each rounded
// up to kUnit values, they are one range that is shared out evenly over warps, not blocks: each warp walks its share
// by itself, so that a few hundred short tensors take a few round trips to memory, not a few hundred.
//
// Squares and sums are float64: a product of two float32 values is exact in it, none overflows, and a sum of 10^9
// loses nothing that float32 could show.  The conversions take 36% of their unit's rate from float32, 63% from bf16.
// Equal calls give equal bits.
// 361 float32 tensors of 27.4 million values into others: 55 us, 21 for the norm (5.2 TB/s), 34 for the rest; one
// bf16 buffer of as many values into a float32 one 38, 13 and 25.  In place, past the limit: 45 float32, 27 bf16.
#include <algorithm>
#include <cfloat>
#include <memory>
#include <new>

#include "common.cuh"
#include "tcgen05.cuh"

namespace rfdetr {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipBlocksPerSm = 4;
constexpr int kUnit = 1024;       // values that a tensor counts for at least
constexpr int kShare = 256;       // a warp's share is a multiple of this
constexpr int kMostTensors = 1000;  // of one launch, whose arguments have 32,764 bytes at most

struct ClipTensor {
    const void *in;
    void *out;
    long long start;  // the tensor's place in the range, times four; plus 1 where the input is bf16, plus 2 where the
                      // output is
    long long count;
};
template <int N> struct ClipTable {
    ClipTensor t[N];
};

struct ClipArgs {
    int n;
    long long total;  // of all tensors, each rounded up
    long long share;  // of a warp
};

struct ClipSums {
    double *sums;    // of all launches' blocks
    int first, all;  // this launch's first; how many there are
};

// The tensor in which place `at` of the whole range lies.
template <int N> __device__ __forceinline__ int tensor_at(const ClipTable<N> &table, int n, long long at) {
    int lo = 0;
#pragma unroll 1
    while (n > 1) {
        const int half = n >> 1;
        const bool before = (table.t[lo + half].start >> 2) <= at;
        lo += before ? half : 0;
        n = before ? n - half : half;
    }
    return lo;
}

// How many values come before the first that lies on 16 bytes.
template <typename T> __device__ __forceinline__ long long ahead_of(const T *p, long long n) {
    const long long k = (16 - (int)(reinterpret_cast<uintptr_t>(p) & 15)) % 16 / (int)sizeof(T);
    return k < n ? k : n;
}

template <typename T> __device__ __forceinline__ void add_square(double &sum, T x) {
    const double v = (double)to_f32(x);
    sum = fma(v, v, sum);
}

// A warp's sum of squares of n values from p.
template <typename T> __device__ __forceinline__ double squares(const T *p, long long n) {
    constexpr int V = 16 / sizeof(T), U = 8;
    const int lane = threadIdx.x & 31;
    double sum[2] = {0.0, 0.0};
    const long long head = ahead_of(p, n);
    if (lane < head) add_square(sum[0], p[lane]);
    const uint4 *body = reinterpret_cast<const uint4 *>(p + head);
    const long long pieces = (n - head) / V, done = head + pieces * V;
#pragma unroll 1
    for (long long i = lane; i < pieces; i += 32 * U) {
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = i + u * 32 < pieces ? __ldg(body + i + u * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) add_square(sum[e & 1], reinterpret_cast<const T *>(&x[u])[e]);
    }
    if (done + lane < n) add_square(sum[1], p[done + lane]);
    return sum[0] + sum[1];
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipBlocksPerSm)
gradient_norm_kernel(const __grid_constant__ ClipTable<N> table, const ClipArgs A, const ClipSums s) {
    __shared__ double part[kClipThreads / 32];
    const int warp = threadIdx.x >> 5;
    long long at = ((long long)blockIdx.x * (kClipThreads / 32) + warp) * A.share;
    const long long end = min(A.total, at + A.share);
    double sum = 0.0;
    launch_dependents();
    if (at < end) {
        int i = tensor_at(table, A.n, at);
#pragma unroll 1
        for (; i < A.n && at < end; ++i) {
            const ClipTensor &t = table.t[i];
            const long long from = at - (t.start >> 2), stop = min(t.count, end - (t.start >> 2));
            if (from < stop)
                sum += t.start & 1 ? squares(static_cast<const bf16 *>(t.in) + from, stop - from)
                                   : squares(static_cast<const float *>(t.in) + from, stop - from);
            at = (t.start >> 2) + (t.count + kUnit - 1) / kUnit * kUnit;
        }
    }
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) part[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < kClipThreads / 32; ++w) all += part[w];
        s.sums[s.first + blockIdx.x] = all;
    }
}

// A warp's n values from p, times f, to q; the last pieces first.  A piece is 16 bytes of the wider of the two types,
// so that a warp's loads and its stores lie together (bf16 to float32 in pieces of 16 bytes of bf16, two stores each:
// 41 us for 27 million values, cold; so: 28).
template <typename T, typename Q> __device__ __forceinline__ void scaled(const T *p, Q *q, long long n, float f) {
    constexpr int V = 16 / (sizeof(T) > sizeof(Q) ? sizeof(T) : sizeof(Q)), U = sizeof(T) * V < 16 ? 8 : 4;
    using In = typename Raw<V * (int)sizeof(T)>::T;
    const int lane = threadIdx.x & 31;
    const long long head = ahead_of(p, n);
    if ((reinterpret_cast<uintptr_t>(q + head) & (V * sizeof(Q) - 1)) == 0) {
        const In *body = reinterpret_cast<const In *>(p + head);
        const long long pieces = (n - head) / V, done = head + pieces * V;
        if (done + lane < n) q[done + lane] = from_f32<Q>(to_f32(p[done + lane]) * f);
#pragma unroll 1
        for (long long i = pieces - 1 - lane; i >= 0; i -= 32 * U) {
            In x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = i - u * 32 >= 0 ? __ldcs(body + i - u * 32) : In{};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i - u * 32 < 0) continue;
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = to_f32(reinterpret_cast<const T *>(&x[u])[e]) * f;
                store_vec<Q, V>(q + head + (i - u * 32) * V, y);
            }
        }
        if (lane < head) q[lane] = from_f32<Q>(to_f32(p[lane]) * f);
        return;
    }
    // Input and output do not lie alike: value by value, lanes side by side.
#pragma unroll 1
    for (long long i = n - 1 - lane; i >= 0; i -= 32 * 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = i - u * 32 >= 0 ? to_f32(p[i - u * 32]) : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i - u * 32 >= 0) q[i - u * 32] = from_f32<Q>(x[u] * f);
    }
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipBlocksPerSm)
gradient_scale_kernel(const __grid_constant__ ClipTable<N> table, const ClipArgs A, const ClipSums s, double limit,
                      float *norm_out) {
    __shared__ double part[kClipThreads / 32];
    const int warp = threadIdx.x >> 5;
    const long long first = ((long long)blockIdx.x * (kClipThreads / 32) + warp) * A.share;
    const long long end = min(A.total, first + A.share);
    int i = first < end ? tensor_at(table, A.n, end - 1) : -1;
    wait_for_primary();
    double sum = 0.0;
    for (int k = threadIdx.x; k < s.all; k += kClipThreads) sum += __ldcg(s.sums + k);
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) part[warp] = sum;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kClipThreads / 32; ++w) all += part[w];
    const double norm = sqrt(all);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float f = norm <= limit ? 1.0f : (float)(limit / norm);
#pragma unroll 1
    for (; i >= 0; --i) {
        const ClipTensor &t = table.t[i];
        const long long start = t.start >> 2;
        const long long from = max(0ll, first - start), n = min(t.count, end - start) - from;
        const int kind = (int)(t.start & 3);
        // In place and within the limit there is nothing to write.
        if (n > 0 && !(f == 1.0f && t.in == t.out)) {
            const float *pf = static_cast<const float *>(t.in) + from;
            const bf16 *pb = static_cast<const bf16 *>(t.in) + from;
            float *qf = static_cast<float *>(t.out) + from;
            bf16 *qb = static_cast<bf16 *>(t.out) + from;
            if (kind == 0) scaled(pf, qf, n, f);
            else if (kind == 1) scaled(pb, qf, n, f);
            else if (kind == 2) scaled(pf, qb, n, f);
            else scaled(pb, qb, n, f);
        }
        if (start <= first) break;
    }
}

// Shares, and blocks, of a launch over `total` values.
struct ClipPlan {
    int blocks;
    long long share;
};
ClipPlan clip_plan(long long total, int sms) {
    constexpr int kWarps = kClipThreads / 32;
    const long long most = (long long)sms * kClipBlocksPerSm * kWarps;
    long long share = (total + most - 1) / most;
    share = share < kUnit ? kUnit : (share + kShare - 1) / kShare * kShare;
    const long long warps = (total + share - 1) / share;
    return {(int)((warps + kWarps - 1) / kWarps), share};
}

long long rounded(long long count) { return (count + kUnit - 1) / kUnit * kUnit; }

struct ClipCall {
    const void *const *in;
    void *const *out;
    const int64_t *counts;
    const int32_t *in_types, *out_types;
};

// Addresses of a tensor's bytes.
struct ClipSpan {
    uintptr_t from, to;
};
ClipSpan span_of(const void *p, int type, int64_t count) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return {at, at + (uintptr_t)count * dtype_size(type)};
}

// Refuses results that share memory with one another, or with a gradient that is not their own: the second launch would
// read what it has written.  Lists in the order of their addresses (a flat buffer's views) take one look at each
// tensor, others a sort; 361 shuffled tensors' call takes 8 to 10 us up to here, in order 6.
int check_memory(const ClipCall &c, int64_t n) {
    const std::unique_ptr<ClipSpan[]> room(new (std::nothrow) ClipSpan[n + 1]);
    if (!room) return RFDETR_ERR_CAPACITY;
    ClipSpan *const spans = room.get();
    int64_t k = 0;
    bool in_order = true;
    for (int64_t i = 0; i < n; ++i) {
        if (c.counts[i] == 0) continue;
        spans[k] = span_of(c.out[i], c.out_types[i], c.counts[i]);
        in_order = in_order && (k == 0 || spans[k - 1].to <= spans[k].from);
        ++k;
    }
    if (!in_order) {
        std::sort(spans, spans + k, [](const ClipSpan &a, const ClipSpan &b) { return a.from < b.from; });
        for (int64_t i = 1; i < k; ++i)
            if (spans[i - 1].to > spans[i].from) return RFDETR_ERR_SHAPE;
    }
    for (int64_t i = 0; i < n; ++i) {
        if (c.counts[i] == 0 || (c.in[i] == c.out[i] && c.in_types[i] == c.out_types[i])) continue;
        const ClipSpan in = span_of(c.in[i], c.in_types[i], c.counts[i]);
        if (in.to <= spans[0].from || in.from >= spans[k - 1].to) continue;
        // The last result that begins before the gradient's end must not reach past its start.
        const ClipSpan *next = std::lower_bound(spans, spans + k, in.to,
                                                [](const ClipSpan &s, uintptr_t end) { return s.from < end; });
        if (next > spans && next[-1].to > in.from) return RFDETR_ERR_SHAPE;
    }
    return RFDETR_OK;
}

// The tensors that have values, from `from` on, up to N of them; returns where the next table begins.
template <int N> int64_t fill_table(ClipTable<N> &table, ClipArgs &A, const ClipCall &c, int64_t from, int64_t n) {
    A = {};
    for (; from < n && A.n < N; ++from) {
        if (c.counts[from] == 0) continue;
        table.t[A.n++] = {c.in[from], c.out[from],
                          A.total * 4 + (c.in_types[from] == RFDETR_BF16) + 2 * (c.out_types[from] == RFDETR_BF16),
                          c.counts[from]};
        A.total += rounded(c.counts[from]);
    }
    return from;
}

template <int N>
int launch_clip(const ClipCall &c, int64_t n, double limit, float *norm, double *sums, cudaStream_t stream) {
    const int sms = num_sms();
    ClipTable<N> table;
    ClipArgs A;
    ClipSums s{sums, 0, 0};
    for (int64_t at = 0; at < n || s.all == 0;) {
        at = fill_table(table, A, c, at, n);
        const ClipPlan p = clip_plan(A.total, sms);
        A.share = p.share;
        s.first = s.all;
        const int blocks = p.blocks > 0 ? p.blocks : 1;  // without values still one, for a norm of 0
        gradient_norm_kernel<N><<<blocks, kClipThreads, 0, stream>>>(table, A, s);
        if (int st = launch_status()) return st;
        s.all += blocks;
    }
    // The launch right after the norms' overlaps their end; it waits for them before it reads or writes anything.
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.blockDim = dim3(kClipThreads);
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    bool first = true;
    for (int64_t at = 0; at < n || first;) {
        if (!first || n > N) at = fill_table(table, A, c, at, n);
        else at = n;  // one table: as the norm's launch had it
        const ClipPlan p = clip_plan(A.total, sms);
        A.share = p.share;
        config.gridDim = dim3((unsigned)(p.blocks > 0 ? p.blocks : 1));
        if (cudaLaunchKernelEx(&config, gradient_scale_kernel<N>, table, A, s, limit, first ? norm : nullptr) !=
            cudaSuccess) {
            (void)cudaGetLastError();
            return RFDETR_ERR_CUDA;
        }
        config.numAttrs = 0;
        first = false;
    }
    return RFDETR_OK;
}

}  // namespace
}  // namespace rfdetr

extern "C" size_t rfdetr_clip_gradients_workspace_bytes(int64_t n_tensors) {
    using namespace rfdetr;
    if (n_tensors < 0 || n_tensors > (1ll << 24)) return 0;
    // A sum for each block of each launch; a launch has four blocks to an SM at most, rounded up once.
    const int64_t tables = n_tensors / kMostTensors + 1;
    return (size_t)tables * (kClipBlocksPerSm * num_sms() + 1) * sizeof(double);
}

extern "C" int rfdetr_clip_gradients(void *stream, const void *const *gradients, const int32_t *gradient_types,
                                     void *const *outputs, const int32_t *output_types, const int64_t *counts,
                                     int64_t n_tensors, double max_norm, float *norm, void *workspace,
                                     size_t workspace_bytes) {
    using namespace rfdetr;
    if (n_tensors < 0 || n_tensors > (1ll << 24) || !(max_norm >= 0.0)) return RFDETR_ERR_SHAPE;
    if (n_tensors > 0 && (!gradients || !gradient_types || !outputs || !output_types || !counts))
        return RFDETR_ERR_SHAPE;
    long long total = 0;
    for (int64_t i = 0; i < n_tensors; ++i) {
        const int in = dtype_size(gradient_types[i]), out = dtype_size(output_types[i]);
        if (in == 0 || out == 0) return RFDETR_ERR_DTYPE;
        if (counts[i] < 0 || counts[i] > (1ll << 40)) return RFDETR_ERR_SHAPE;
        total += rounded(counts[i]);
        if (total > (1ll << 42)) return RFDETR_ERR_SHAPE;
        if (counts[i] && (!gradients[i] || !outputs[i] || !aligned(gradients[i], in) || !aligned(outputs[i], out)))
            return RFDETR_ERR_ALIGN;
        if (counts[i] && gradients[i] == outputs[i] && in != out) return RFDETR_ERR_DTYPE;
    }
    if (!norm || !aligned(norm, 4)) return RFDETR_ERR_ALIGN;
    const ClipCall c{gradients, outputs, counts, gradient_types, output_types};
    if (int st = check_memory(c, n_tensors)) return st;
    if (!workspace || workspace_bytes < rfdetr_clip_gradients_workspace_bytes(n_tensors) || !aligned(workspace, 8))
        return RFDETR_ERR_WORKSPACE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double *sums = static_cast<double *>(workspace);
    // The arguments are copied at every launch: a short list takes a short table.
    if (n_tensors <= 32) return launch_clip<32>(c, n_tensors, max_norm, norm, sums, s);
    if (n_tensors <= 384) return launch_clip<384>(c, n_tensors, max_norm, norm, sums, s);
    return launch_clip<kMostTensors>(c, n_tensors, max_norm, norm, sums, s);
}
