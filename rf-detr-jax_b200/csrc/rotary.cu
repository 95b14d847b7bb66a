// Rotary positions with several axes, for queries and keys in one launch.
//
// Frequency i of R/2 belongs to an axis a(i) (consecutive sections, one per axis) and turns the
// pair (x1, x2) of every head of token t by theta = positions[t, a(i)] * inv_freq[i]:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
// with (x1, x2) the channels (i, i + R/2), or (2i, 2i + 1) when interleaved; channels from R on are
// copied.  The gradient is the same turn by -theta.
//
// The bound is memory: each value is read and written once, and the turns are a few operations on
// it.  So that the sines stay out of the way, a block takes a few tokens, forms their cosines and
// sines once in shared memory for all heads of q and k, and then streams the heads through in
// 16-byte pieces.  The angle is formed in float64 and reduced to a fraction of a turn before it is
// narrowed: at position 16384 a float32 product is already wrong by 1e-3 radians.
#include "common.cuh"

namespace rfdetr {
namespace {

constexpr int kMaxAxes = 8;
constexpr int kRotaryThreads = 256;
constexpr double kInvTwoPi = 0.15915494309189533576888;

struct RotaryArgs {
    const void *in[2];       // q, k
    void *out[2];            // contiguous [T, H, D]
    long long token[2], head[2];  // input strides, elements
    int heads[2];
    const void *positions;   // [T, n_axes]
    const float *inv_freq;   // [half]
    int ends[kMaxAxes];      // end of each axis's section of frequencies
    int n_axes;
    long long T;
    int D, half;
    int per_block;           // tokens
    Divisor per_token, per_head, half_of;  // pieces of a token and of a head; half
    float sign;              // -1: the inverse turn
};

// The turned pair, its products and sums fused the same way whatever the piece: results do not depend on
// an input's alignment.
__device__ __forceinline__ float first_of(float x1, float x2, float2 r) {
    return __fmaf_rn(x1, r.x, -__fmul_rn(x2, r.y));
}
__device__ __forceinline__ float second_of(float x1, float x2, float2 r) {
    return __fmaf_rn(x2, r.x, __fmul_rn(x1, r.y));
}

// Pieces of VEC channels.  A head's pieces: the turned ones first (one piece of x1 and one of x2,
// or one piece of VEC / 2 pairs), then the copied ones.  A thread asks for its first piece before the
// sines are formed, so that their time covers the load's.  32,768 tokens of 20 x 128 channels, bf16, take 54 us
// (6.2 TB/s, 96% of the measured copy rate), 20,011 of 8 x 80, partly turned, 25.8 there and back; with a
// second piece in flight per thread 3 us more and 0.7 less.  Places are found with known divisors (57.6 and 31.0
// us by division).

// Where frequency i's cosine and sine are: one place is left out after every piece's, so that the pieces of a warp's
// lanes read from different banks (without: 7 us more for the first of the tokens above).
template <int VEC, bool INTERLEAVED> __host__ __device__ constexpr int turn_at(int i) {
    constexpr int kGroup = INTERLEAVED ? VEC / 2 : VEC;
    return kGroup > 1 ? i + i / kGroup : i;
}

template <typename T, typename P, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) axial_rotary_kernel(const RotaryArgs A) {
    using V = typename Raw<VEC * (int)sizeof(T)>::T;
    extern __shared__ float2 turn[];  // [token][turn_at(half)]
    const int pitch = turn_at<VEC, INTERLEAVED>(A.half);
    const long long t0 = (long long)blockIdx.x * A.per_block;
    const int tokens = (int)min((long long)A.per_block, A.T - t0);
    const int R = 2 * A.half;
    const int turned = (INTERLEAVED ? R : A.half) / VEC;
    const int pieces = tokens * A.per_token.d;

    struct Piece {
        T *out;
        int token, c;
        bool turns;
        V x1, x2;
    } p;
    auto ask = [&](int x) {
        const int t = quotient(x, A.per_token), y = x - t * A.per_token.d;
        int h = quotient(y, A.per_head);
        const int piece = y - h * A.per_head.d;
        const int which = h >= A.heads[0];
        h -= which ? A.heads[0] : 0;
        const T *in = static_cast<const T *>(A.in[which]) + (t0 + t) * A.token[which] + h * A.head[which];
        p.turns = piece < turned;
        p.c = p.turns ? piece * VEC : R + (piece - turned) * VEC;
        p.token = t;
        p.out = static_cast<T *>(A.out[which]) + ((t0 + t) * A.heads[which] + h) * A.D + p.c;
        p.x1 = __ldg(reinterpret_cast<const V *>(in + p.c));
        if (!INTERLEAVED && p.turns) p.x2 = __ldg(reinterpret_cast<const V *>(in + p.c + A.half));
    };
    if ((int)threadIdx.x < pieces) ask(threadIdx.x);

    const P *pos = static_cast<const P *>(A.positions) + t0 * A.n_axes;
    for (int x = threadIdx.x; x < tokens * A.half; x += kRotaryThreads) {
        const int t = quotient(x, A.half_of), i = x - t * A.half;
        int axis = 0;
        while (i >= A.ends[axis]) ++axis;
        const double turns = (double)pos[t * A.n_axes + axis] * (double)__ldg(A.inv_freq + i) * kInvTwoPi;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[t * pitch + turn_at<VEC, INTERLEAVED>(i)] = make_float2(c, s * A.sign);
    }
    __syncthreads();

    for (int x = threadIdx.x; x < pieces;) {
        if (p.turns) {
            const float2 *cs = turn + p.token * pitch + turn_at<VEC, INTERLEAVED>(INTERLEAVED ? p.c / 2 : p.c);
            const T *a = reinterpret_cast<const T *>(&p.x1), *b = reinterpret_cast<const T *>(&p.x2);
            float u[VEC], w[VEC];
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 r = cs[e >> 1];
                    const float x1 = to_f32(a[e]), x2 = to_f32(a[e + 1]);
                    u[e] = first_of(x1, x2, r);
                    u[e + 1] = second_of(x1, x2, r);
                }
                store_vec<T, VEC>(p.out, u);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 r = cs[e];
                    const float x1 = to_f32(a[e]), x2 = to_f32(b[e]);
                    u[e] = first_of(x1, x2, r);
                    w[e] = second_of(x1, x2, r);
                }
                store_vec<T, VEC>(p.out, u);
                store_vec<T, VEC>(p.out + A.half, w);
            }
        } else {
            *reinterpret_cast<V *>(p.out) = p.x1;
        }
        x += kRotaryThreads;
        if (x < pieces) ask(x);
    }
}

template <typename T, typename P, int VEC>
int launch_rotary(const RotaryArgs &A, bool interleaved, cudaStream_t stream) {
    const long long blocks = (A.T + A.per_block - 1) / A.per_block;
    if (blocks > 0x7fffffffll) return RFDETR_ERR_SHAPE;
    auto smem = [&](int pitch) { return (size_t)A.per_block * pitch * sizeof(float2); };
    if (interleaved) {
        if constexpr (VEC >= 2)
            axial_rotary_kernel<T, P, VEC, true>
                <<<(unsigned)blocks, kRotaryThreads, smem(turn_at<VEC, true>(A.half)), stream>>>(A);
        else
            return RFDETR_ERR_SHAPE;
    } else {
        axial_rotary_kernel<T, P, VEC, false>
            <<<(unsigned)blocks, kRotaryThreads, smem(turn_at<VEC, false>(A.half)), stream>>>(A);
    }
    return launch_status();
}

template <typename T, typename P>
int dispatch_rotary(const RotaryArgs &A, bool interleaved, int vec, cudaStream_t stream) {
    if (vec * sizeof(T) >= 16) return launch_rotary<T, P, 16 / sizeof(T)>(A, interleaved, stream);
    if (vec >= 2) return launch_rotary<T, P, 2>(A, interleaved, stream);
    return launch_rotary<T, P, 1>(A, interleaved, stream);
}

}  // namespace
}  // namespace rfdetr

extern "C" int rfdetr_axial_rotary(void *stream, const void *query, int64_t query_token_stride,
                                   int64_t query_head_stride, const void *key, int64_t key_token_stride,
                                   int64_t key_head_stride, int dtype, const void *positions, int position_dtype,
                                   const float *inv_freq, const int64_t *sections, int64_t n_axes, void *query_out,
                                   void *key_out, int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
                                   int64_t head_dim, int interleaved, int inverse) {
    using namespace rfdetr;
    if (dtype_size(dtype) == 0 ||
        (position_dtype != RFDETR_F32 && position_dtype != RFDETR_I32 && position_dtype != RFDETR_I64))
        return RFDETR_ERR_DTYPE;
    if (tokens < 0 || tokens > (1ll << 40) || n_heads < 0 || n_heads > 65536 || n_kv_heads < 0 || n_kv_heads > 65536 ||
        head_dim < 2 || head_dim > 1024 || n_axes < 1 || n_axes > kMaxAxes || !sections)
        return RFDETR_ERR_SHAPE;
    if (query_token_stride < 0 || query_head_stride < 0 || key_token_stride < 0 || key_head_stride < 0)
        return RFDETR_ERR_SHAPE;
    RotaryArgs A{};
    long long half = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0 || sections[a] > head_dim) return RFDETR_ERR_SHAPE;
        half += sections[a];
        A.ends[a] = (int)half;
    }
    if (half < 1 || 2 * half > head_dim) return RFDETR_ERR_SHAPE;
    if (n_kv_heads == 0) key = query, key_out = query_out;  // not read or written
    if (tokens == 0 || n_heads + n_kv_heads == 0) return RFDETR_OK;
    const int size = dtype_size(dtype);
    if ((n_heads && (!query || !query_out || !aligned(query, size) || !aligned(query_out, size))) ||
        (n_kv_heads && (!key || !key_out || !aligned(key, size) || !aligned(key_out, size))) || !positions ||
        !aligned(positions, position_dtype == RFDETR_I64 ? 8 : 4) || !inv_freq || !aligned(inv_freq, 4))
        return RFDETR_ERR_ALIGN;
    A.in[0] = query, A.in[1] = key, A.out[0] = query_out, A.out[1] = key_out;
    A.token[0] = query_token_stride, A.token[1] = key_token_stride;
    A.head[0] = query_head_stride, A.head[1] = key_head_stride;
    A.heads[0] = (int)n_heads, A.heads[1] = (int)n_kv_heads;
    A.positions = positions, A.inv_freq = inv_freq, A.n_axes = (int)n_axes;
    A.T = tokens, A.D = (int)head_dim, A.half = (int)half, A.sign = inverse ? -1.0f : 1.0f;
    // The widest piece, up to 16 bytes, that every address and boundary allows.
    int vec = 16 / size;
    auto fits = [&](int v) {
        const long long b = (long long)v * size;
        bool ok = head_dim % v == 0 && (interleaved ? 2 * half : half) % v == 0;
        for (int w = 0; w < 2; ++w)
            if (A.heads[w])
                ok = ok && aligned(A.in[w], b) && aligned(A.out[w], b) && A.token[w] % v == 0 && A.head[w] % v == 0;
        return ok;
    };
    if (!fits(vec)) vec = fits(2) ? 2 : 1;
    if (interleaved && vec < 2) return RFDETR_ERR_ALIGN;
    // Tokens to a block: two pieces to a thread (one: 69.7 us for the first of the tokens above and 29.0 for the
    // second; four: 53.5 and 26.6; eight: 56.9 and 28.5), fewer where that would leave SMs without four blocks, and no more than 16 KB of sines.
    const long long turned = interleaved ? 2 * half / vec : half / vec;
    const long long per_head = turned + (head_dim - 2 * half) / vec;
    const long long per_token = per_head * (n_heads + n_kv_heads);
    A.per_head = divisor((int)per_head), A.per_token = divisor((int)per_token), A.half_of = divisor((int)half);
    long long per = 2ll * kRotaryThreads / per_token;
    const long long spread = tokens / (4ll * num_sms()), most = 16384 / (half * (long long)sizeof(float2));
    per = per > spread ? spread : per;
    per = per > most ? most : per;
    A.per_block = (int)(per < 1 ? 1 : per);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool il = interleaved != 0;
    auto with = [&](auto element) {
        using T = decltype(element);
        if (position_dtype == RFDETR_F32) return dispatch_rotary<T, float>(A, il, vec, s);
        if (position_dtype == RFDETR_I32) return dispatch_rotary<T, int32_t>(A, il, vec, s);
        return dispatch_rotary<T, int64_t>(A, il, vec, s);
    };
    return dtype == RFDETR_BF16 ? with(bf16{}) : with(float{});
}
