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
// The floor is memory: forward x in and y out, backward x and g in and dx out; nothing is kept between them.  What
// bounds it now is the issue of instructions, 64% of the slots forward and 54% backward: 32,768 tokens of 16 + 4 heads
// of 128, bf16, take 73 and 129 us, 4.6 and 3.9 TB/s; 20,011 of 7 + 1 of 80, 48 channels interleaved, 14.4 and 28.2;
// float32, 8192 of 16 + 4 of 256, 64 turned, 93 and 181, 3.6 and 2.8 TB/s.  A row (one head of one token) is read once,
// in 16-byte pieces, by as many neighbouring lanes as it has pieces, or half as many (normed_plan.cuh; ten for 80
// channels of bf16, three rows to a warp), summed by shuffles, and turned in registers.  Where half is a multiple
// of a piece a lane holds both partners of its pairs; otherwise they meet through shared memory, so that any half is
// read in whole pieces.  Blocks stay for the launch: a lane's channels are the same in every row, so the weights'
// gradients are summed in its registers, then over the block, and a second launch adds the blocks' sums in order (no
// atomics: equal calls give equal bits).  Sums, norms and angles are float32 (angles reduced from a product carried
// twice as far); values are rounded to the output's type once.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "normed_plan.cuh"
#include "tcgen05.cuh"

namespace rfdetr {
namespace {

constexpr int kAxes = 8;
constexpr int kNormThreads = 256, kNormWarps = kNormThreads / 32;
constexpr int kMostDim = 256;
constexpr double kTurnsPerRadian = 0.15915494309189533576888;

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
    bool full;                    // no lane of a row lacks a piece, or a piece its second vector
    int per_chunk;                // tokens that share a forming of sines
    int sines_at_once;            // of them, by the threads of a block
    int pieces, lanes;            // of a row; lanes that hold it
    Divisor lanes_of, half_of;
    float eps, inv_dim;
    float *partial;               // backward: [blocks][2][D], or null
};

// A position times a frequency (radians per unit), in turns, reduced to half a turn at most.  Where the position is a
// float and the turns are below 2^22 the frequency in turns and the product are each carried as two floats, good
// to 2^-46 of the product; otherwise, and to the same end, float64.
__device__ __forceinline__ float turns_of(const NormArgs &A, long long at, float inv_freq) {
    constexpr float kHigh = (float)kTurnsPerRadian, kLow = (float)(kTurnsPerRadian - (double)kHigh);
    float p;
    double far;
    bool exact = true;
    if (A.position_type == RFDETR_F32) {
        p = __ldg(static_cast<const float *>(A.positions) + at);
        far = (double)p;
    } else if (A.position_type == RFDETR_I32) {
        const int32_t v = __ldg(static_cast<const int32_t *>(A.positions) + at);
        p = (float)v;
        far = (double)v;
        exact = v > -(1 << 24) && v < 1 << 24;
    } else {
        const long long v = __ldg(static_cast<const long long *>(A.positions) + at);
        p = (float)v;
        far = (double)v;
        exact = v > -(1 << 24) && v < 1 << 24;
    }
    const float f = __fmul_rn(inv_freq, kHigh), low = fmaf(inv_freq, kLow, fmaf(inv_freq, kHigh, -f));
    const float turns = __fmul_rn(p, f);
    if (exact && fabsf(turns) < 4194304.0f)
        return __fsub_rn(turns, rintf(turns)) + fmaf(p, low, fmaf(p, f, -turns));
    const double all = far * (double)inv_freq * kTurnsPerRadian;
    return (float)(all - rint(all));
}

// Places in shared memory: one is left out after every VEC, so that lanes' pieces lie in different banks.
template <int VEC> __host__ __device__ constexpr int spread(int i) { return VEC > 1 ? i + i / VEC : i; }

// The sum over the lanes of a row, in each of them; `at` is the lane's place in the row.
__device__ __forceinline__ float row_sum(float x, int at, int lanes) {
    if ((lanes & (lanes - 1)) == 0) {
#pragma unroll
        for (int o = 1; o < 32; o *= 2)
            if (o < lanes) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        if (o >= lanes) break;
        const float y = __shfl_down_sync(0xffffffffu, x, o);
        x += at + o < lanes ? y : 0.0f;
    }
    return __shfl_sync(0xffffffffu, x, (threadIdx.x & 31) - at);
}

// 1 / sqrt(x), the hardware's approximation and a step of Newton's: within an ulp or so.
__device__ __forceinline__ float inverse_root(float x) {
    const float r = rsqrtf(x);
    const float e = fmaf(-x * r, r, 1.0f);
    return x > 0.0f && x <= FLT_MAX ? fmaf(0.5f * r, e, r) : r;  // (0 and inf: their roots' inverses as they are)
}

// A lane's row, a head of a token of one of the two tensors, and its way to the next of its rows in a chunk.
template <typename T> struct Row {
    const T *x, *g;
    T *y;
    int h, token;  // tokens from the chunk's first on
    bool live;
};
struct Stride {
    int t, h, y;  // tokens and heads on (heads past the last are the next token's), and elements of the output
    long long x, g, wrap_x, wrap_g;
};

template <bool BACK> __device__ __forceinline__ Stride stride_of(const NormArgs &A, int which, int step) {
    Stride s;
    const int heads = A.heads[which];
    s.t = quotient(step, A.heads_of[which]);
    s.h = step - s.t * heads;
    s.y = step * A.D;
    s.x = s.t * A.token[which] + s.h * A.head[which];
    s.wrap_x = A.token[which] - heads * A.head[which];
    s.g = BACK ? s.t * A.grad_token[which] + s.h * A.grad_head[which] : 0;
    s.wrap_g = BACK ? A.grad_token[which] - heads * A.grad_head[which] : 0;
    return s;
}
template <typename T, bool BACK>
__device__ __forceinline__ Row<T> row_of(const NormArgs &A, int which, long long t0, int row, bool live) {
    Row<T> r;
    row = live ? row : 0;
    r.token = quotient(row, A.heads_of[which]);
    r.h = row - r.token * A.heads[which];
    r.live = live;
    const long long t = t0 + r.token;
    r.x = static_cast<const T *>(A.in[which]) + t * A.token[which] + r.h * A.head[which];
    r.g = BACK ? static_cast<const T *>(A.grad[which]) + t * A.grad_token[which] + r.h * A.grad_head[which] : nullptr;
    r.y = static_cast<T *>(A.out[which]) + (t0 * A.heads[which] + row) * A.D;
    return r;
}
template <typename T, bool BACK> __device__ __forceinline__ void go_on(Row<T> &r, const Stride &s, int heads) {
    r.token += s.t;
    r.h += s.h;
    r.x += s.x;
    if (BACK) r.g += s.g;
    r.y += s.y;
    if (r.h >= heads) {
        r.h -= heads;
        ++r.token;
        r.x += s.wrap_x;
        if (BACK) r.g += s.wrap_g;
    }
}

// VEC values to 16-byte-aligned memory; bf16 rounded two at a time.
template <typename T, int VEC> __device__ __forceinline__ void put_values(T *p, const float *x) {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int e = 0; e < VEC; e += 2) w[e / 2] = pack_bf16(x[e], x[e + 1]);
        using V = typename Raw<VEC * 2>::T;
        *reinterpret_cast<V *>(p) = *reinterpret_cast<V *>(w);
    } else {
        store_vec<T, VEC>(p, x);
    }
}

// N of float32 pairs from and to 16-byte-aligned shared memory, as wide as they go.
template <int N> __device__ __forceinline__ void load_pairs(const float *p, int stride4, float2 *v) {
    if constexpr (N == 1) {
        v[0] = *reinterpret_cast<const float2 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float4 x = *reinterpret_cast<const float4 *>(p + (i / 2) * stride4);
            v[i] = make_float2(x.x, x.y);
            v[i + 1] = make_float2(x.z, x.w);
        }
    }
}

// Rows whose lanes hold both partners of their pairs.  A lane has N pieces of P pairs of channels, as float32 pairs
// (of neighbouring channel pairs) of first partners and of second: packed arithmetic takes half the issue slots (with
// scalar arithmetic, and places found by division for every row, the first of the sizes above took 95 us forward and
// 167 backward).  In shared memory cosines and sines, and weights, lie by pieces: four pairs' of all pieces, then the
// next four.
template <typename T, int VEC, int MODE, int N, bool BACK> struct PairRows {
    static constexpr int P = MODE == kPaired ? VEC : VEC / 2, Q = P / 2;  // pairs, float2 of them
    static constexpr int K = MODE == kPaired ? 2 : 1;
    using V = typename Raw<VEC * (int)sizeof(T)>::T;
    struct Values {
        float2 a[N][Q], b[N][Q];
    };
    struct Raws {
        V x[N][K], g[BACK ? N : 1][K];
    };
    // What is the same for every row.
    struct Lane {
        int c[N];        // first channel, elements; paired: of the first vector
        bool has[N], turns[N];
    };

    static __device__ __forceinline__ Lane lane_of(const NormArgs &A, int at) {
        Lane l;
        const int turned = MODE == kPaired ? A.half / VEC : (2 * A.half + VEC - 1) / VEC;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int piece = at + n * A.lanes;
            l.has[n] = piece < A.pieces;
            l.turns[n] = piece < turned;
            l.c[n] = MODE != kPaired || l.turns[n] ? piece * VEC : 2 * A.half + (piece - turned) * VEC;
        }
        return l;
    }
    // Shared memory: floats of a token's cosines and sines, of a weight, and where a channel's or pair's value goes.
    static __host__ __device__ int turn_floats(const NormArgs &A) { return 2 * ((A.half + P - 1) / P * P); }
    static __host__ __device__ int row_floats(const NormArgs &A) { return (2 * A.pieces * P + 3) / 4 * 4; }
    static __device__ __forceinline__ int by_pieces(int i, int pieces) {  // of value i, P to a piece
        if (P < 4) return i;
        return ((i % P / 4) * pieces + i / P) * 4 + i % 4;
    }
    static __device__ __forceinline__ int turn_place(const NormArgs &A, int i) {
        return by_pieces(i, (A.half + P - 1) / P);
    }
    // Of channel c in a weight's row: first partners, then second ones.
    static __device__ __forceinline__ int weight_place(const NormArgs &A, int c) {
        const int all = A.pieces * P;
        if (MODE == kInterleaved) return (c & 1) * all + by_pieces(c >> 1, A.pieces);
        const int R = 2 * A.half, turned = A.half / VEC;
        if (c >= R) return by_pieces(turned * P + c - R, A.pieces);
        return c >= A.half ? all + by_pieces(c - A.half, A.pieces) : by_pieces(c, A.pieces);
    }
    static __device__ __forceinline__ void weights(const NormArgs &A, const float *w, int piece, float2 *a, float2 *b) {
        constexpr int kPlace = P < 4 ? P : 4;
        load_pairs<Q>(w + piece * kPlace, A.pieces * 4, a);
        load_pairs<Q>(w + A.pieces * P + piece * kPlace, A.pieces * 4, b);
    }

    static __device__ __forceinline__ void load(const NormArgs &A, const Lane &l, const Row<T> &w, Raws &r) {
        // Every lane of a row has all of its vectors (a row that is none reads another one's, for nothing).
        if (A.full) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    r.x[n][k] = __ldg(reinterpret_cast<const V *>(w.x + l.c[n] + k * A.half));
                    if (BACK) r.g[n][k] = __ldg(reinterpret_cast<const V *>(w.g + l.c[n] + k * A.half));
                }
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const bool ok = w.live && l.has[n] && (k == 0 || l.turns[n]);
                const int c = l.c[n] + k * A.half;
                r.x[n][k] = ok ? __ldg(reinterpret_cast<const V *>(w.x + c)) : V{};
                if (BACK) r.g[n][k] = ok ? __ldg(reinterpret_cast<const V *>(w.g + c)) : V{};
            }
    }
    static __device__ __forceinline__ float wide(const V &v, int e) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(&v)[e / 2];
            return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
        } else {
            return to_f32(reinterpret_cast<const T *>(&v)[e]);
        }
    }
    static __device__ __forceinline__ void widen(const V (&raw)[N][K], Values &v) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                if (MODE == kPaired) {
                    v.a[n][i] = make_float2(wide(raw[n][0], 2 * i), wide(raw[n][0], 2 * i + 1));
                    v.b[n][i] = make_float2(wide(raw[n][K - 1], 2 * i), wide(raw[n][K - 1], 2 * i + 1));
                } else {
                    v.a[n][i] = make_float2(wide(raw[n][0], 4 * i), wide(raw[n][0], 4 * i + 2));
                    v.b[n][i] = make_float2(wide(raw[n][0], 4 * i + 1), wide(raw[n][0], 4 * i + 3));
                }
            }
    }
    template <bool INVERSE>
    static __device__ __forceinline__ void turned(const NormArgs &A, const Lane &l, int at, Values &v,
                                                  const float *turn) {
        const float2 minus = make_float2(-1.0f, -1.0f);
        const int pieces = (A.half + P - 1) / P;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (!l.turns[n]) continue;
            float2 c[Q], s[Q];
            constexpr int kPlace = P < 4 ? P : 4;
            load_pairs<Q>(turn + (at + n * A.lanes) * kPlace, pieces * 4, c);
            load_pairs<Q>(turn + pieces * P + (at + n * A.lanes) * kPlace, pieces * 4, s);
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float2 x = v.a[n][i], y = v.b[n][i], xs = mul2(x, s[i]), ys = mul2(y, s[i]);
                float2 u = INVERSE ? fma2(x, c[i], ys) : fma2(x, c[i], mul2(ys, minus));
                float2 w = INVERSE ? fma2(y, c[i], mul2(xs, minus)) : fma2(y, c[i], xs);
                if (MODE == kInterleaved && A.half % P != 0) {  // of the last piece some do not turn
                    const int pair = l.c[n] / 2 + 2 * i;
                    if (pair >= A.half) u.x = x.x, w.x = y.x;
                    if (pair + 1 >= A.half) u.y = x.y, w.y = y.y;
                }
                v.a[n][i] = u;
                v.b[n][i] = w;
            }
        }
    }
    static __device__ __forceinline__ void store(const NormArgs &A, const Lane &l, T *y, const Values &v, float r,
                                                 bool live) {
        const float2 r2 = make_float2(r, r);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (!live || !l.has[n]) continue;
            float x[K][VEC];
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float2 u = mul2(v.a[n][i], r2), w = mul2(v.b[n][i], r2);
                if (MODE == kPaired) {
                    x[0][2 * i] = u.x, x[0][2 * i + 1] = u.y;
                    x[K - 1][2 * i] = w.x, x[K - 1][2 * i + 1] = w.y;
                } else {
                    x[0][4 * i] = u.x, x[0][4 * i + 2] = u.y;
                    x[0][4 * i + 1] = w.x, x[0][4 * i + 3] = w.y;
                }
            }
            put_values<T, VEC>(y + l.c[n], x[0]);
            if (MODE == kPaired && l.turns[n]) put_values<T, VEC>(y + l.c[n] + A.half, x[K - 1]);
        }
    }
    static __device__ __forceinline__ float square(const Values &v) {
        float2 sum = make_float2(0.0f, 0.0f), more = sum;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                sum = fma2(v.a[n][i], v.a[n][i], sum);
                more = fma2(v.b[n][i], v.b[n][i], more);
            }
        return (sum.x + sum.y) + (more.x + more.y);
    }

    // A row from its raw values to its result; backward adds to the weights' gradient.  Whole warp.
    static __device__ __forceinline__ void row(const NormArgs &A, const Lane &l, const Raws &raw, T *y, bool live,
                                               int at, const float *weight, const float *turn, float *, Values &dw) {
        Values x;
        widen(raw.x, x);
        const float sum = square(x);
        if (!BACK) {
            const float r = inverse_root(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (!l.has[n]) continue;
                float2 wa[Q], wb[Q];
                weights(A, weight, at + n * A.lanes, wa, wb);
#pragma unroll
                for (int i = 0; i < Q; ++i) {
                    x.a[n][i] = mul2(x.a[n][i], wa[i]);
                    x.b[n][i] = mul2(x.b[n][i], wb[i]);
                }
            }
            turned<false>(A, l, at, x, turn);
            store(A, l, y, x, r, live);
            return;
        }
        Values g;
        if constexpr (BACK) widen(raw.g, g);
        turned<true>(A, l, at, g, turn);
        Values wh;
        float2 dot = make_float2(0.0f, 0.0f), more = dot;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float2 wa[Q], wb[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) wa[i] = wb[i] = make_float2(0.0f, 0.0f);
            if (l.has[n]) weights(A, weight, at + n * A.lanes, wa, wb);
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                wh.a[n][i] = mul2(g.a[n][i], wa[i]);
                wh.b[n][i] = mul2(g.b[n][i], wb[i]);
                dot = fma2(wh.a[n][i], x.a[n][i], dot);
                more = fma2(wh.b[n][i], x.b[n][i], more);
            }
        }
        const float r = inverse_root(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
        const float back = -(row_sum((dot.x + dot.y) + (more.x + more.y), at, A.lanes) * A.inv_dim * r * r);
        const float2 back2 = make_float2(back, back), r2 = make_float2(r, r);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                wh.a[n][i] = fma2(x.a[n][i], back2, wh.a[n][i]);
                wh.b[n][i] = fma2(x.b[n][i], back2, wh.b[n][i]);
                x.a[n][i] = mul2(x.a[n][i], r2);
                x.b[n][i] = mul2(x.b[n][i], r2);
            }
        if (live) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < Q; ++i) {
                    dw.a[n][i] = fma2(g.a[n][i], x.a[n][i], dw.a[n][i]);
                    dw.b[n][i] = fma2(g.b[n][i], x.b[n][i], dw.b[n][i]);
                }
        }
        store(A, l, y, wh, r, live);
    }
    // A lane's sums of dw to its row of shared memory, where the weights' values have their places.
    static __device__ __forceinline__ void put(const NormArgs &A, const Lane &l, int at, const Values &v, float *to) {
        constexpr int kPlace = P < 4 ? P : 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (!l.has[n]) continue;
            const int piece = at + n * A.lanes;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int place = (i / 4) * A.pieces * 4 + piece * kPlace + i % 4;
                to[place] = i & 1 ? v.a[n][i / 2].y : v.a[n][i / 2].x;
                to[A.pieces * P + place] = i & 1 ? v.b[n][i / 2].y : v.b[n][i / 2].x;
            }
        }
    }
};

// Rows whose partners meet through shared memory; a lane has N pieces of VEC channels.
template <typename T, int VEC, int N, bool BACK> struct ExchangeRows {
    using V = typename Raw<VEC * (int)sizeof(T)>::T;
    using Values = float[N][VEC];
    struct Raws {
        V x[N], g[BACK ? N : 1];
    };
    struct Lane {
        int at;
    };

    static __device__ __forceinline__ Lane lane_of(const NormArgs &, int at) { return {at}; }
    static __host__ __device__ int turn_floats(const NormArgs &A) { return 2 * (spread<VEC>(A.half) + 1); }
    static __host__ __device__ int row_floats(const NormArgs &A) { return spread<VEC>(A.D) + 1; }
    static __device__ __forceinline__ int turn_place(const NormArgs &, int i) { return spread<VEC>(i); }
    static __device__ __forceinline__ int weight_place(const NormArgs &, int c) { return spread<VEC>(c); }

    static __device__ __forceinline__ void load(const NormArgs &A, const Lane &l, const Row<T> &w, Raws &r) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int piece = l.at + n * A.lanes;
            const bool ok = w.live && piece < A.pieces;
            r.x[n] = ok ? __ldg(reinterpret_cast<const V *>(w.x + piece * VEC)) : V{};
            if (BACK) r.g[n] = ok ? __ldg(reinterpret_cast<const V *>(w.g + piece * VEC)) : V{};
        }
    }
    static __device__ __forceinline__ void widen(const V (&raw)[N], Values &v) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[n][e] = to_f32(reinterpret_cast<const T *>(&raw[n])[e]);
    }
    // Whole warp.
    template <bool INVERSE>
    static __device__ __forceinline__ void turned(const NormArgs &A, Values &v, int at, bool live, const float *turn,
                                                  float *room) {
        const int R = 2 * A.half;
        __syncwarp();  // the row before has been read
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int c = (at + n * A.lanes) * VEC + e;
                if (live && c < R) room[spread<VEC>(c)] = v[n][e];
            }
        __syncwarp();
        if (!live) return;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int d = (at + n * A.lanes) * VEC + e;
                if (d >= R) continue;
                const bool first = A.interleaved ? !(d & 1) : d < A.half;
                const int other = A.interleaved ? d ^ 1 : first ? d + A.half : d - A.half;
                const float *cs = turn + spread<VEC>(A.interleaved ? d >> 1 : first ? d : other);
                const float s = cs[spread<VEC>(A.half) + 1];
                v[n][e] = fmaf(v[n][e], cs[0], room[spread<VEC>(other)] * (first != INVERSE ? -s : s));
            }
    }
    static __device__ __forceinline__ void store(const NormArgs &A, T *y, int at, Values &v, bool live) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (live && at + n * A.lanes < A.pieces) put_values<T, VEC>(y + (at + n * A.lanes) * VEC, v[n]);
    }
    static __device__ __forceinline__ void row(const NormArgs &A, const Lane &, const Raws &raw, T *y, bool live,
                                               int at, const float *weight, const float *turn, float *room, Values &dw) {
        Values x;
        widen(raw.x, x);
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(x[n][e], x[n][e], sum);
        if (!BACK) {
            const float r = inverse_root(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const float *w = weight + spread<VEC>((at + n * A.lanes) * VEC);
                const bool ok = at + n * A.lanes < A.pieces;
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[n][e] *= r * (ok ? w[e] : 0.0f);
            }
            turned<false>(A, x, at, live, turn, room);
            store(A, y, at, x, live);
            return;
        }
        Values g, wh;
        if constexpr (BACK) widen(raw.g, g);
        turned<true>(A, g, at, live, turn, room);
        float dot = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float *w = weight + spread<VEC>((at + n * A.lanes) * VEC);
            const bool ok = at + n * A.lanes < A.pieces;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                wh[n][e] = g[n][e] * (ok ? w[e] : 0.0f);
                dot = fmaf(wh[n][e], x[n][e], dot);
            }
        }
        const float r = inverse_root(fmaf(row_sum(sum, at, A.lanes), A.inv_dim, A.eps));
        const float back = row_sum(dot, at, A.lanes) * A.inv_dim * r * r;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                wh[n][e] = r * fmaf(-x[n][e], back, wh[n][e]);
                if (live) dw[n][e] = fmaf(g[n][e], x[n][e] * r, dw[n][e]);
            }
        store(A, y, at, wh, live);
    }
    static __device__ __forceinline__ void put(const NormArgs &A, const Lane &, int at, const Values &v, float *to) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (at + n * A.lanes < A.pieces)
#pragma unroll
                for (int e = 0; e < VEC; ++e) to[spread<VEC>((at + n * A.lanes) * VEC) + e] = v[n][e];
    }
};

template <typename T, int VEC, int MODE, int N, bool BACK>
using RowsOf = std::conditional_t<MODE == kExchange, ExchangeRows<T, VEC, N, BACK>,
                                  PairRows<T, VEC, MODE == kExchange ? kPaired : MODE, N, BACK>>;

// Floats of shared memory: sines, both weights, and the exchange's rows or the sums of dw.
template <typename S, bool EXCHANGE> struct NormRoom {
    int pitch, row, sines, all;
    __host__ __device__ NormRoom(const NormArgs &A, bool back) {
        pitch = S::turn_floats(A);
        sines = (A.per_chunk * pitch + 3) / 4 * 4;
        row = S::row_floats(A);
        const int rows = kNormWarps * (32 / A.lanes);
        all = sines + 2 * row + (back || EXCHANGE ? rows * row : 0);
    }
};

template <bool BACK> constexpr int kNormBlocks = BACK ? 2 : 3;  // to an SM

template <typename T, int VEC, int MODE, int N, bool BACK>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks<BACK>) normed_rotary_kernel(const NormArgs A) {
    using S = RowsOf<T, VEC, MODE, N, BACK>;
    extern __shared__ __align__(16) float turn[];
    const NormRoom<S, MODE == kExchange> room(A, BACK);
    float *weights = turn + room.sines;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows_a_warp = 32 / A.lanes;
    const int sub = quotient(lane, A.lanes_of), at = lane - sub * A.lanes;
    const bool used = sub < rows_a_warp;
    float *mine = weights + 2 * room.row + (warp * rows_a_warp + min(sub, rows_a_warp - 1)) * room.row;
    const int step = kNormWarps * rows_a_warp;  // rows from one of a lane's to the next
    const typename S::Lane place = S::lane_of(A, at);

    typename S::Values dw[BACK ? 2 : 1] = {};
#pragma unroll 1
    for (long long chunk = blockIdx.x; chunk < A.chunks; chunk += gridDim.x) {
        const long long t0 = chunk * A.per_chunk;
        const int tokens = (int)min((long long)A.per_chunk, A.T - t0);
        // The first row is asked for before the sines are formed, so that their time covers the load's, and
        // each further one before the one before is worked on.
        const int start = warp * rows_a_warp;
        typename S::Raws ahead;
        Row<T> next;
        auto ask = [&](int which) {
            next = row_of<T, BACK>(A, which, t0, start + sub, used && start + sub < tokens * A.heads[which]);
            S::load(A, place, next, ahead);
        };
        if (start < tokens * A.heads[0]) ask(0);
        __syncthreads();
        if (chunk == blockIdx.x) {
            for (int i = threadIdx.x; i < 2 * room.row; i += kNormThreads) weights[i] = 0.0f;  // (places of no channel)
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * A.D; i += kNormThreads) {
                const int which = i >= A.D, c = i - which * A.D;
                const void *w = A.weight[which];
                weights[which * room.row + S::weight_place(A, c)] =
                    !w ? 1.0f
                       : A.weight_type[which] == RFDETR_BF16 ? to_f32(static_cast<const bf16 *>(w)[c])
                                                             : static_cast<const float *>(w)[c];
            }
        }
        // A thread keeps to one frequency.
        const int first = quotient(threadIdx.x, A.half_of), i = threadIdx.x - first * A.half;
        if (first < A.sines_at_once) {
            int axis = 0;
            while (i >= A.ends[axis]) ++axis;
            const float inv_freq = __ldg(A.inv_freq + i);
            float *cs = turn + first * room.pitch + S::turn_place(A, i);
#pragma unroll 1
            for (int t = first; t < tokens; t += A.sines_at_once) {
                float s, c;
                sincospif(2.0f * turns_of(A, (t0 + t) * A.n_axes + axis, inv_freq), &s, &c);
                cs[0] = c;
                cs[room.pitch / 2] = s;
                cs += A.sines_at_once * room.pitch;
            }
        }
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int rows = tokens * A.heads[which];
            if (which == 1 && start < rows) ask(1);
            const Stride stride = stride_of<BACK>(A, which, step);
#pragma unroll 1
            for (int x = start; x < rows; x += step) {
                const typename S::Raws raw = ahead;
                T *const to = next.y;
                const bool live = next.live;
                const float *cs = turn + (live ? next.token : 0) * room.pitch;
                if (x + step < rows) {
                    next.live = used && x + step + sub < rows;
                    if (next.live) go_on<T, BACK>(next, stride, A.heads[which]);  // else it stays at a row that is
                    S::load(A, place, next, ahead);
                }
                S::row(A, place, raw, to, live, at, weights + which * room.row, cs, mine, dw[BACK ? which : 0]);
            }
        }
    }
    if constexpr (BACK) {
        launch_dependents();
        if (!A.partial) return;
        float *sums = weights + 2 * room.row;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (used) S::put(A, place, at, dw[which], mine);
            __syncthreads();
            for (int c = threadIdx.x; c < A.D; c += kNormThreads) {
                float sum = 0.0f;
                for (int r = 0; r < kNormWarps * rows_a_warp; ++r) sum += sums[r * room.row + S::weight_place(A, c)];
                A.partial[((size_t)blockIdx.x * 2 + which) * A.D + c] = sum;
            }
        }
    }
}

// The blocks' sums of dw, 32 columns to a block, added in order.
constexpr int kSumRows = 32;
__global__ void __launch_bounds__(32 * kSumRows)
weight_grad_kernel(const float *partial, int blocks, int D, void *dwq, int q_type, void *dwk, int k_type) {
    __shared__ float part[kSumRows][33];
    const int column = blockIdx.x * 32 + threadIdx.x;
    wait_for_primary();
    float sum = 0.0f;
    if (column < 2 * D) {
#pragma unroll 8
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
int launch_normed(NormArgs &A, const NormPlan &plan, const WeightGrads &dw, cudaStream_t stream) {
    // A row lies within a warp: with more lanes the kernel's step from row to row would be 0.
    if (plan.lanes < 1 || plan.lanes > 32 || plan.each != N || plan.mode != MODE || plan.vec != VEC)
        return RFDETR_ERR_SHAPE;
    A.pieces = plan.pieces;
    A.lanes = plan.lanes;
    A.lanes_of = divisor(A.lanes);
    A.full = MODE != kExchange && A.pieces == A.lanes * N && (MODE != kPaired || 2 * A.half == A.D);
    // Tokens that share a forming of sines: eight rows to a lane, no more than 16 KB of sines, and of those as many as
    // give every block that stays the same number of chunks (20,011 tokens of 8 x 80: 445 chunks for 444 blocks took
    // 19.8 us).
    constexpr int kBlocks = kNormBlocks<BACK>;
    static_assert(!BACK || kBlocks <= kBackBlocks, "the workspace");
    const long long stay = kBlocks * (long long)num_sms();
    const int at_once = kNormWarps * (32 / A.lanes);
    const long long one = at_once / (A.heads[0] + A.heads[1]), most = 16384 / (A.half * (long long)sizeof(float2));
    long long per = 8 * one > 1 ? 8 * one : 1;
    per = per > most ? most : per;
    const long long rounds = (A.T + per * stay - 1) / (per * stay);
    const long long even = (A.T + rounds * stay - 1) / (rounds * stay);
    per = even > one ? even : one;  // (a row to a lane at least)
    per = per > most ? most : per;
    A.per_chunk = (int)(per < 1 ? 1 : per);
    A.sines_at_once = kNormThreads / A.half;  // half is 128 at most
    A.chunks = (A.T + A.per_chunk - 1) / A.per_chunk;
    const size_t bytes =
        NormRoom<RowsOf<T, VEC, MODE, N, BACK>, MODE == kExchange>(A, BACK).all * sizeof(float);
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

template <typename T, bool BACK>
int dispatch_normed(NormArgs &A, bool whole, const WeightGrads &dw, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const NormPlan p = plan_normed(sizeof(T), A.D, A.half, A.interleaved, whole);
    if (!whole) return launch_normed<T, 1, kExchange, 8, BACK>(A, p, dw, stream);
    switch (p.mode) {
        case kInterleaved: return launch_normed<T, V, kInterleaved, 2, BACK>(A, p, dw, stream);
        case kExchange: return launch_normed<T, V, kExchange, 2, BACK>(A, p, dw, stream);
        default: break;
    }
    if constexpr (V == 4)
        if (p.each == 2) return launch_normed<T, V, kPaired, 2, BACK>(A, p, dw, stream);
    return launch_normed<T, V, kPaired, 1, BACK>(A, p, dw, stream);
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
