// The root-mean-square norm of every head of queries and keys, and rotary positions with several axes on the result,
// in one pass:
//   r = 1 / sqrt(mean_c x_c^2 + eps),  n_c = x_c r w_c,  y = R(theta) n
// with R the turn of axial_rotary (rotary.cu): frequency i turns a pair of channels, (i, i + half) or, interleaved,
// (2i, 2i + 1), by theta = positions[t, a(i)] inv_freq[i]; channels from 2 half on are normed only.  With the
// cotangent g of y, h = R(-theta) g:
//   dw_c = sum over tokens and heads of h_c x_c r,
//   dx_c = r (w_c h_c - x_c r^2 mean_c' (w_c' h_c' x_c'))
// r is formed again from x, which the gradient reads anyway.
//
// The bound is memory: forward x in and y out, backward x and g in and dx out; nothing is kept between them.  A row
// (one head of one token) is read once, in 16-byte pieces, by as many neighbouring lanes as it has pieces (ten for 80
// channels of bf16, three rows to a warp), summed by shuffles, and turned in registers.  Where half is a
// multiple of a piece a lane holds both partners of its pairs; otherwise they meet through shared memory, so that any
// half is read in whole pieces.  Blocks stay for the launch: a lane's channels are the same in every row,
// so the weights' gradients are summed in its registers, then over the block, and a second launch adds the blocks' sums
// in order (no atomics: equal calls give equal bits).
// Sums, norms and angles are float32 (angles reduced in float64); values are rounded to the output's type once.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace rfdetr {
namespace {

constexpr int kAxes = 8;
constexpr int kNormThreads = 256, kNormWarps = kNormThreads / 32;
constexpr int kMostDim = 256;
constexpr double kTurnsPerRadian = 0.15915494309189533576888;

// How a lane finds the partners of its channels: it holds both (paired, interleaved), or through shared memory.
enum { kPaired, kInterleaved, kExchange };

struct NormArgs {
    const void *in[2];            // q, k
    const void *grad[2];          // backward: their outputs' cotangents
    void *out[2];                 // contiguous [T, H, D]
    const void *weight[2];        // [D] or null
    long long token[2], head[2];  // strides, elements
    long long grad_token[2], grad_head[2];
    int heads[2];
    Divisor heads_of[2];
    int weight_type[2];
    const void *positions;        // [T, n_axes]
    int position_type;
    const float *inv_freq;        // [half]
    int ends[kAxes];              // end of each axis's section of frequencies
    int n_axes;
    long long T, chunks;
    int D, half;
    bool interleaved;
    int per_chunk;                // tokens that share a forming of sines
    int pieces, lanes;            // of a row; lanes that hold it
    Divisor lanes_of, half_of;
    float eps, inv_dim;
    float *partial;               // backward: [blocks][2][D], or null
};

__device__ __forceinline__ double position_at(const NormArgs &A, long long i) {
    if (A.position_type == RFDETR_I32) return (double)static_cast<const int32_t *>(A.positions)[i];
    if (A.position_type == RFDETR_I64) return (double)static_cast<const int64_t *>(A.positions)[i];
    return (double)static_cast<const float *>(A.positions)[i];
}

// Places in shared memory: one is left out after every VEC, so that lanes' pieces lie in different banks.
template <int VEC> __host__ __device__ constexpr int spread(int i) { return VEC > 1 ? i + i / VEC : i; }

// The sum over the lanes of a row, in each of them; `at` is the lane's place in the row.
__device__ __forceinline__ float row_sum(float x, int at, int lanes) {
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        if (o >= lanes) break;
        const float y = __shfl_down_sync(0xffffffffu, x, o);
        x += at + o < lanes ? y : 0.0f;
    }
    return __shfl_sync(0xffffffffu, x, (threadIdx.x & 31) - at);
}

// N pieces to a lane (the row's pieces at, at + lanes, ...), each of K vectors of VEC channels.
template <typename T, int VEC, int MODE, int N, bool BACK> struct Rows {
    static constexpr int K = MODE == kPaired ? 2 : 1;
    using V = typename Raw<VEC * (int)sizeof(T)>::T;
    using Values = float[N][K][VEC];

    struct Raws {
        V x[N][K], g[BACK ? N : 1][K];
    };

    // First channel of vector k of a piece, and whether there is such a vector.
    static __device__ __forceinline__ int channel(const NormArgs &A, int piece, int k) {
        if (MODE != kPaired) return piece * VEC;
        const int turned = A.half / VEC;
        return piece < turned ? piece * VEC + k * A.half : 2 * A.half + (piece - turned) * VEC;
    }
    static __device__ __forceinline__ bool has(const NormArgs &A, int piece, int k) {
        return piece < A.pieces && (MODE != kPaired || k == 0 || piece < A.half / VEC);
    }

    static __device__ __forceinline__ void load(const NormArgs &A, int which, long long t, int h, int at, bool live,
                                                Raws &r) {
        const T *x = static_cast<const T *>(A.in[which]) + t * A.token[which] + h * A.head[which];
        const T *g = BACK ? static_cast<const T *>(A.grad[which]) + t * A.grad_token[which] + h * A.grad_head[which]
                          : nullptr;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int piece = at + n * A.lanes;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const bool ok = live && has(A, piece, k);
                const int c = channel(A, piece, k);
                r.x[n][k] = ok ? __ldg(reinterpret_cast<const V *>(x + c)) : V{};
                if (BACK) r.g[n][k] = ok ? __ldg(reinterpret_cast<const V *>(g + c)) : V{};
            }
        }
    }
    static __device__ __forceinline__ void widen(const V (&raw)[N][K], Values &v) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[n][k][e] = to_f32(reinterpret_cast<const T *>(&raw[n][k])[e]);
    }

    // Turns a row's values; `turn` holds the token's cosines and sines, `room` a row for the exchange.  Whole warp.
    template <int SIGN>
    static __device__ __forceinline__ void turned(const NormArgs &A, Values &v, int at, bool live, const float2 *turn,
                                                  float *room) {
        const int R = 2 * A.half;
        if (MODE == kExchange) {
            __syncwarp();  // the row before has been read
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int c = channel(A, at + n * A.lanes, 0) + e;
                    if (live && c < R) room[spread<VEC>(c)] = v[n][0][e];
                }
            __syncwarp();
        }
        if (!live) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int piece = at + n * A.lanes, c = channel(A, piece, 0);
            if (MODE == kPaired) {
                if (!has(A, piece, K - 1)) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 r = turn[spread<VEC>(c) + e];
                    const float x1 = v[n][0][e], x2 = v[n][K - 1][e], s = SIGN * r.y;
                    v[n][0][e] = fmaf(x1, r.x, -(x2 * s));
                    v[n][K - 1][e] = fmaf(x2, r.x, x1 * s);
                }
            } else if (MODE == kInterleaved) {
#pragma unroll
                for (int e = 0; e + 1 < VEC; e += 2) {
                    if (c + e >= R) continue;
                    const float2 r = turn[spread<VEC / 2>((c + e) / 2)];
                    const float x1 = v[n][0][e], x2 = v[n][0][e + 1], s = SIGN * r.y;
                    v[n][0][e] = fmaf(x1, r.x, -(x2 * s));
                    v[n][0][e + 1] = fmaf(x2, r.x, x1 * s);
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int d = c + e;
                    if (d >= R) continue;
                    const bool first = A.interleaved ? !(d & 1) : d < A.half;
                    const int other = A.interleaved ? d ^ 1 : first ? d + A.half : d - A.half;
                    const float2 r = turn[spread<VEC>(A.interleaved ? d >> 1 : first ? d : other)];
                    const float s = first ? -SIGN * r.y : SIGN * r.y;
                    v[n][0][e] = fmaf(v[n][0][e], r.x, room[spread<VEC>(other)] * s);
                }
            }
        }
    }

    static __device__ __forceinline__ void store(const NormArgs &A, const Values &v, int which, long long t, int h,
                                                 int at, bool live) {
        T *y = static_cast<T *>(A.out[which]) + (t * A.heads[which] + h) * A.D;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (live && has(A, at + n * A.lanes, k))
                    store_vec<T, VEC>(y + channel(A, at + n * A.lanes, k), v[n][k]);
    }

    // A row from its raw values to its result; backward adds to the weights' gradient.  Whole warp.
    static __device__ __forceinline__ void row(const NormArgs &A, const Raws &raw, int which, long long t, int h,
                                               int at, bool live, const float *weight, const float2 *turn, float *room,
                                               Values &dw) {
        Values x;
        widen(raw.x, x);
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum = fmaf(x[n][k][e], x[n][k][e], sum);
        if (!BACK) {
            const float r = __frsqrt_rn(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float *w = weight + spread<VEC>(channel(A, at + n * A.lanes, k));
                    const bool ok = has(A, at + n * A.lanes, k);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) x[n][k][e] *= r * (ok ? w[e] : 0.0f);
                }
            turned<1>(A, x, at, live, turn, room);
            store(A, x, which, t, h, at, live);
            return;
        }
        Values g;
        if constexpr (BACK) widen(raw.g, g);
        turned<-1>(A, g, at, live, turn, room);
        float dot = 0.0f;
        Values wh;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float *w = weight + spread<VEC>(channel(A, at + n * A.lanes, k));
                const bool ok = has(A, at + n * A.lanes, k);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    wh[n][k][e] = g[n][k][e] * (ok ? w[e] : 0.0f);
                    dot = fmaf(wh[n][k][e], x[n][k][e], dot);
                }
            }
        const float r = __frsqrt_rn(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
        const float back = row_sum(dot, at, A.lanes) * A.inv_dim * r * r;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (live) dw[n][k][e] = fmaf(g[n][k][e], x[n][k][e] * r, dw[n][k][e]);
                    wh[n][k][e] = r * fmaf(-x[n][k][e], back, wh[n][k][e]);
                }
        store(A, wh, which, t, h, at, live);
    }
};

// Floats of shared memory: sines, both weights, and the larger of the exchange's rows and the sums of dw.
template <int VEC, int MODE> struct NormRoom {
    static constexpr int kGroup = MODE == kInterleaved ? VEC / 2 : VEC;
    int pitch, weights, row, sines, all;
    __host__ __device__ NormRoom(const NormArgs &A, bool back) {
        pitch = spread<kGroup>(A.half) + 1;
        sines = 2 * A.per_chunk * pitch;
        row = spread<VEC>(A.D) + 1;
        weights = 2 * row;
        const int rows = kNormWarps * (32 / A.lanes);
        all = sines + weights + (back || MODE == kExchange ? rows * row : 0);
    }
};

template <typename T, int VEC, int MODE, int N, bool BACK>
__global__ void __launch_bounds__(kNormThreads, BACK || N == 2 ? 2 : 4) normed_rotary_kernel(const NormArgs A) {
    using S = Rows<T, VEC, MODE, N, BACK>;
    using Room = NormRoom<VEC, MODE>;
    extern __shared__ float2 turn[];
    const Room room(A, BACK);
    float *weights = reinterpret_cast<float *>(turn) + room.sines;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows_a_warp = 32 / A.lanes;
    const int sub = quotient(lane, A.lanes_of), at = lane - sub * A.lanes;
    const bool used = sub < rows_a_warp;
    float *mine = weights + room.weights + (warp * rows_a_warp + min(sub, rows_a_warp - 1)) * room.row;
    constexpr int kStep = kNormWarps;  // rows, times rows_a_warp, from one of a lane's to the next

    typename S::Values dw[BACK ? 2 : 1] = {};
#pragma unroll 1
    for (long long chunk = blockIdx.x; chunk < A.chunks; chunk += gridDim.x) {
        const long long t0 = chunk * A.per_chunk;
        const int tokens = (int)min((long long)A.per_chunk, A.T - t0);
        // The first row is asked for before the sines are formed, so that their time covers the load's.
        typename S::Raws raw;
        auto ask = [&](int which, int x) {
            const int at_row = x + sub, t = quotient(at_row, A.heads_of[which]);
            S::load(A, which, t0 + t, at_row - t * A.heads[which], at, used && at_row < tokens * A.heads[which], raw);
        };
        const int start = warp * rows_a_warp;
        if (start < tokens * A.heads[0]) ask(0, start);
        __syncthreads();
        if (chunk == blockIdx.x) {
            for (int i = threadIdx.x; i < 2 * A.D; i += kNormThreads) {
                const int which = i >= A.D, c = i - which * A.D;
                const void *w = A.weight[which];
                weights[which * room.row + spread<VEC>(c)] =
                    !w ? 1.0f
                       : A.weight_type[which] == RFDETR_BF16 ? to_f32(static_cast<const bf16 *>(w)[c])
                                                             : static_cast<const float *>(w)[c];
            }
        }
        for (int x = threadIdx.x; x < tokens * A.half; x += kNormThreads) {
            const int t = quotient(x, A.half_of), i = x - t * A.half;
            int axis = 0;
            while (i >= A.ends[axis]) ++axis;
            const double turns = position_at(A, (t0 + t) * A.n_axes + axis) * (double)__ldg(A.inv_freq + i) *
                                 kTurnsPerRadian;
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            turn[t * room.pitch + spread<Room::kGroup>(i)] = make_float2(c, s);
        }
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int rows = tokens * A.heads[which];
#pragma unroll 1
            for (int x = start; x < rows; x += kStep * rows_a_warp) {
                if (which == 1 || x != start) ask(which, x);
                const int at_row = x + sub, t = quotient(at_row, A.heads_of[which]);
                const bool live = used && at_row < rows;
                S::row(A, raw, which, t0 + t, at_row - t * A.heads[which], at, live, weights + which * room.row,
                       turn + (live ? t : 0) * room.pitch, mine, dw[BACK ? which : 0]);
            }
        }
    }
    if constexpr (BACK) {
        launch_dependents();
        if (!A.partial) return;
        float *sums = weights + room.weights;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (used)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < S::K; ++k)
                        if (S::has(A, at + n * A.lanes, k))
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                mine[spread<VEC>(S::channel(A, at + n * A.lanes, k)) + e] = dw[which][n][k][e];
            __syncthreads();
            for (int c = threadIdx.x; c < A.D; c += kNormThreads) {
                float sum = 0.0f;
                for (int r = 0; r < kNormWarps * rows_a_warp; ++r) sum += sums[r * room.row + spread<VEC>(c)];
                A.partial[((size_t)blockIdx.x * 2 + which) * A.D + c] = sum;
            }
        }
    }
}

// The blocks' sums of dw, 32 columns to a block, added in order.
constexpr int kSumRows = 16;
__global__ void __launch_bounds__(32 * kSumRows)
weight_grad_kernel(const float *partial, int blocks, int D, void *dwq, int q_type, void *dwk, int k_type) {
    __shared__ float part[kSumRows][33];
    const int column = blockIdx.x * 32 + threadIdx.x;
    wait_for_primary();
    float sum = 0.0f;
    if (column < 2 * D) {
#pragma unroll 4
        for (int b = threadIdx.y; b < blocks; b += kSumRows) sum += __ldcg(partial + (size_t)b * 2 * D + column);
    }
    part[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y > 0 || column >= 2 * D) return;
    sum = 0.0f;
#pragma unroll
    for (int r = 0; r < kSumRows; ++r) sum += part[r][threadIdx.x];
    const int which = column >= D, c = column - which * D;
    void *out = which ? dwk : dwq;
    if (!out) return;
    if ((which ? k_type : q_type) == RFDETR_BF16) static_cast<bf16 *>(out)[c] = from_f32<bf16>(sum);
    else static_cast<float *>(out)[c] = sum;
}

struct WeightGrads {
    void *out[2];
    int type[2];
};

constexpr int kBackBlocks = 2;  // to an SM

template <typename T, int VEC, int MODE, int N, bool BACK>
int launch_normed(NormArgs &A, const WeightGrads &dw, cudaStream_t stream) {
    A.lanes = A.pieces < 32 ? A.pieces : 32;
    A.lanes_of = divisor(A.lanes);
    // Tokens that share a forming of sines: four rows to a lane, fewer where that would leave SMs without
    // work, and no more than 16 KB of sines.
    const int rows = A.heads[0] + A.heads[1], at_once = kNormWarps * (32 / A.lanes);
    long long per = 4ll * at_once / rows;
    const long long spread_out = A.T / ((BACK ? kBackBlocks : 4) * (long long)num_sms());
    const long long most = 16384 / (A.half * (long long)sizeof(float2));
    per = per > spread_out ? spread_out : per;
    per = per > most ? most : per;
    A.per_chunk = (int)(per < 1 ? 1 : per);
    A.chunks = (A.T + A.per_chunk - 1) / A.per_chunk;
    const size_t bytes = NormRoom<VEC, MODE>(A, BACK).all * sizeof(float);
    const long long stay = (BACK ? kBackBlocks : 4) * (long long)num_sms();
    const int blocks = (int)(A.chunks < stay ? A.chunks : stay);
    auto kernel = normed_rotary_kernel<T, VEC, MODE, N, BACK>;
    if (bytes > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
        return RFDETR_ERR_CUDA;
    kernel<<<blocks, kNormThreads, bytes, stream>>>(A);
    if (int st = launch_status()) return st;
    if (!BACK || !A.partial) return RFDETR_OK;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)((2 * A.D + 31) / 32));
    config.blockDim = dim3(32, kSumRows);
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, weight_grad_kernel, (const float *)A.partial, blocks, A.D, dw.out[0], dw.type[0],
                           dw.out[1], dw.type[1]) != cudaSuccess) {
        (void)cudaGetLastError();
        return RFDETR_ERR_CUDA;
    }
    return RFDETR_OK;
}

template <typename T, bool BACK> int dispatch_normed(NormArgs &A, bool whole, const WeightGrads &dw, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (!whole) {  // a value at a time
        A.pieces = A.D;
        return launch_normed<T, 1, kExchange, kMostDim / 32, BACK>(A, dw, stream);
    }
    const bool paired = !A.interleaved && A.half % V == 0;
    A.pieces = paired ? A.half / V + (A.D - 2 * A.half) / V : A.D / V;
    auto with = [&](auto mode) {
        constexpr int M = decltype(mode)::value;
        if constexpr (kMostDim / V > 32) {
            if (A.pieces > 32) return launch_normed<T, V, M, 2, BACK>(A, dw, stream);
        }
        return launch_normed<T, V, M, 1, BACK>(A, dw, stream);
    };
    if (paired) return with(std::integral_constant<int, kPaired>{});
    if (A.interleaved) return with(std::integral_constant<int, kInterleaved>{});
    return with(std::integral_constant<int, kExchange>{});
}

struct NormCall {
    const void *in[2], *grad[2], *weight[2];
    void *out[2];
    int64_t token[2], head[2], grad_token[2], grad_head[2], heads[2];
    int weight_type[2];
    int dtype, position_dtype;
    const void *positions;
    const float *inv_freq;
    const int64_t *sections;
    int64_t n_axes, tokens, head_dim;
    float eps;
    int interleaved;
};

// Checks a call and fills the kernel's arguments; whole: all pieces are of 16 bytes.
int check_normed(const NormCall &c, bool back, NormArgs &A, bool &whole) {
    if (dtype_size(c.dtype) == 0 || dtype_size(c.weight_type[0]) == 0 || dtype_size(c.weight_type[1]) == 0 ||
        (c.position_dtype != RFDETR_F32 && c.position_dtype != RFDETR_I32 && c.position_dtype != RFDETR_I64))
        return RFDETR_ERR_DTYPE;
    if (c.tokens < 0 || c.tokens > (1ll << 40) || c.head_dim < 2 || c.head_dim > kMostDim || c.n_axes < 1 ||
        c.n_axes > kAxes || !c.sections || !(c.eps >= 0.0f) || c.eps > FLT_MAX)
        return RFDETR_ERR_SHAPE;
    long long half = 0;
    for (int a = 0; a < c.n_axes; ++a) {
        if (c.sections[a] < 0 || c.sections[a] > c.head_dim) return RFDETR_ERR_SHAPE;
        half += c.sections[a];
        A.ends[a] = (int)half;
    }
    if (half < 1 || 2 * half > c.head_dim) return RFDETR_ERR_SHAPE;
    const int size = dtype_size(c.dtype), vec = 16 / size;
    whole = c.head_dim % vec == 0;
    for (int w = 0; w < 2; ++w) {
        if (c.heads[w] < 0 || c.heads[w] > 65536 || c.token[w] < 0 || c.head[w] < 0 ||
            (back && (c.grad_token[w] < 0 || c.grad_head[w] < 0)))
            return RFDETR_ERR_SHAPE;
        A.in[w] = c.in[w], A.out[w] = c.out[w], A.weight[w] = c.weight[w], A.weight_type[w] = c.weight_type[w];
        A.token[w] = c.token[w], A.head[w] = c.head[w], A.heads[w] = (int)c.heads[w];
        A.heads_of[w] = divisor(c.heads[w] > 0 ? (int)c.heads[w] : 1);
        if (back) A.grad[w] = c.grad[w], A.grad_token[w] = c.grad_token[w], A.grad_head[w] = c.grad_head[w];
        if (c.heads[w] == 0 || c.tokens == 0) continue;
        if (!c.in[w] || !c.out[w] || !aligned(c.in[w], size) || !aligned(c.out[w], size) ||
            !aligned(c.weight[w], dtype_size(c.weight_type[w])) ||
            (back && (!c.grad[w] || !aligned(c.grad[w], size))))
            return RFDETR_ERR_ALIGN;
        whole = whole && aligned(c.in[w], 16) && aligned(c.out[w], 16) && c.token[w] % vec == 0 &&
                c.head[w] % vec == 0;
        if (back) whole = whole && aligned(c.grad[w], 16) && c.grad_token[w] % vec == 0 && c.grad_head[w] % vec == 0;
    }
    if (c.tokens > 0 && c.heads[0] + c.heads[1] > 0 &&
        (!c.positions || !aligned(c.positions, c.position_dtype == RFDETR_I64 ? 8 : 4) || !c.inv_freq ||
         !aligned(c.inv_freq, 4)))
        return RFDETR_ERR_ALIGN;
    A.positions = c.positions, A.position_type = c.position_dtype, A.inv_freq = c.inv_freq, A.n_axes = (int)c.n_axes;
    A.T = c.tokens, A.D = (int)c.head_dim, A.half = (int)half, A.half_of = divisor((int)half);
    A.interleaved = c.interleaved != 0;
    A.eps = c.eps, A.inv_dim = 1.0f / (float)c.head_dim;
    return RFDETR_OK;
}

}  // namespace
}  // namespace rfdetr

extern "C" int rfdetr_normed_rotary(void *stream, const void *query, int64_t query_token_stride,
                                    int64_t query_head_stride, const void *key, int64_t key_token_stride,
                                    int64_t key_head_stride, int dtype, const void *query_weight,
                                    int query_weight_dtype, const void *key_weight, int key_weight_dtype, float eps,
                                    const void *positions, int position_dtype, const float *inv_freq,
                                    const int64_t *sections, int64_t n_axes, void *query_out, void *key_out,
                                    int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                    int interleaved) {
    using namespace rfdetr;
    const NormCall c{{query, key}, {nullptr, nullptr}, {query_weight, key_weight}, {query_out, key_out},
                     {query_token_stride, key_token_stride}, {query_head_stride, key_head_stride}, {0, 0}, {0, 0},
                     {n_heads, n_kv_heads}, {query_weight_dtype, key_weight_dtype}, dtype, position_dtype, positions,
                     inv_freq, sections, n_axes, tokens, head_dim, eps, interleaved};
    NormArgs A{};
    bool whole = false;
    if (int st = check_normed(c, false, A, whole)) return st;
    if (tokens == 0 || n_heads + n_kv_heads == 0) return RFDETR_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == RFDETR_BF16 ? dispatch_normed<bf16, false>(A, whole, {}, s)
                                : dispatch_normed<float, false>(A, whole, {}, s);
}

extern "C" size_t rfdetr_normed_rotary_backward_workspace_bytes(int64_t head_dim) {
    using namespace rfdetr;
    if (head_dim < 2 || head_dim > kMostDim) return 0;
    return (size_t)kBackBlocks * num_sms() * 2 * head_dim * sizeof(float);
}

extern "C" int rfdetr_normed_rotary_backward(
    void *stream, const void *query, int64_t query_token_stride, int64_t query_head_stride, const void *key,
    int64_t key_token_stride, int64_t key_head_stride, const void *grad_query_out, int64_t grad_query_token_stride,
    int64_t grad_query_head_stride, const void *grad_key_out, int64_t grad_key_token_stride,
    int64_t grad_key_head_stride, int dtype, const void *query_weight, int query_weight_dtype, const void *key_weight,
    int key_weight_dtype, float eps, const void *positions, int position_dtype, const float *inv_freq,
    const int64_t *sections, int64_t n_axes, void *grad_query, void *grad_key, void *grad_query_weight,
    void *grad_key_weight, void *workspace, size_t workspace_bytes, int64_t tokens, int64_t n_heads,
    int64_t n_kv_heads, int64_t head_dim, int interleaved) {
    using namespace rfdetr;
    const NormCall c{{query, key}, {grad_query_out, grad_key_out}, {query_weight, key_weight}, {grad_query, grad_key},
                     {query_token_stride, key_token_stride}, {query_head_stride, key_head_stride},
                     {grad_query_token_stride, grad_key_token_stride}, {grad_query_head_stride, grad_key_head_stride},
                     {n_heads, n_kv_heads}, {query_weight_dtype, key_weight_dtype}, dtype, position_dtype, positions,
                     inv_freq, sections, n_axes, tokens, head_dim, eps, interleaved};
    NormArgs A{};
    bool whole = false;
    if (int st = check_normed(c, true, A, whole)) return st;
    if (!aligned(grad_query_weight, dtype_size(query_weight_dtype)) ||
        !aligned(grad_key_weight, dtype_size(key_weight_dtype)))
        return RFDETR_ERR_ALIGN;
    const bool weights = grad_query_weight || grad_key_weight;
    if (weights && (!workspace || !aligned(workspace, 4) ||
                    workspace_bytes < rfdetr_normed_rotary_backward_workspace_bytes(head_dim)))
        return RFDETR_ERR_WORKSPACE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tokens == 0 || n_heads + n_kv_heads == 0) {  // sums of nothing
        void *const out[2] = {grad_query_weight, grad_key_weight};
        const int types[2] = {query_weight_dtype, key_weight_dtype};
        for (int w = 0; w < 2; ++w)
            if (out[w] && cudaMemsetAsync(out[w], 0, head_dim * dtype_size(types[w]), s) != cudaSuccess)
                return RFDETR_ERR_CUDA;
        return RFDETR_OK;
    }
    A.partial = weights ? static_cast<float *>(workspace) : nullptr;
    const WeightGrads dw{{grad_query_weight, grad_key_weight}, {query_weight_dtype, key_weight_dtype}};
    return dtype == RFDETR_BF16 ? dispatch_normed<bf16, true>(A, whole, dw, s)
                                : dispatch_normed<float, true>(A, whole, dw, s);
}
