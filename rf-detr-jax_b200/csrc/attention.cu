// Softmax attention over packed sequences, forward and backward, on the tensor cores (tcgen05).
//
// For sequence s with Lq queries and Lk keys, query i of head h and key j of head h / G:
//   S_ij = scale q_i.k_j,  lse_i = log sum_j exp S_ij,  P_ij = exp(S_ij - lse_i),  o_i = sum_j P_ij v_j
// over the keys that i may see: all, or with `causal` those with j <= i + Lk - Lq.  A query that
// sees none has o_i = 0 and lse_i = -inf.  With the cotangent g of o (and c of lse):
//   dP_ij = g_i.v_j,  delta_i = o_i.g_i - c_i,  dS_ij = P_ij (dP_ij - delta_i),
//   dV_j = sum_i P_ij g_i,  dK_j = scale sum_i dS_ij q_i,  dQ_i = scale sum_j dS_ij k_j
// (dK, dV summed over the G query heads of a key head).
//
// Sequences are ranges of rows of q and of k/v, given by offsets on the device.  A block finds its
// rows from its index alone: sequence x owns the tile slots from start(x) / R + x on (R rows to a
// slot), which never overlap and always suffice, so no plan has to be made and no length has to be
// known on the host.  The rows before the first and after the last sequence count as sequences
// without keys: their outputs and gradients are zero.  Offsets are clamped to the tensors.
// Scores are float32: a row whose scores are all -inf has no weights and is treated as one that sees no key.
//
// Queries of the heads that share a key head are rows of one tile (token-major, heads inner), so
// K and V are read once for all of them and a few tokens still fill a tile.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace rfdetr {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const int32_t *q_off, *k_off;  // [n_seq + 1]
    int n_seq, Tq, Tk;
    int Hq, Hkv, D;
    int pack;    // query heads in one tile (of those that share a key head)
    int pack_inv;  // 65536 / pack rounded up: row / pack for rows up to 255
    int subs;    // tiles' head groups per key head: (Hq / Hkv) / pack
    int causal;
    float scale, scale_log2;
    Divisor slot_rows;  // rows (of the tensor that the launch tiles) in a slot
    Divisor heads;      // key heads x head groups: blocks or row tiles to a slot
};

// A tile row's token within the tile and its head among the packed ones.
__device__ __forceinline__ int row_token(const AttnArgs &A, int row) { return (row * A.pack_inv) >> 16; }
__device__ __forceinline__ int row_head(const AttnArgs &A, int row) { return row - row_token(A, row) * A.pack; }

// Bytes of a tile row panel and panels per row, for channels padded to DP.
template <int DP> struct Tile {
    static constexpr int kRowBytes = DP == 32 ? 64 : 128;
    static constexpr int kPanels = DP * 2 / kRowBytes;
    static constexpr int kCols = kRowBytes / 2;  // channels in a panel
};

__device__ __forceinline__ int off_at(const int32_t *off, int n_seq, int T, int x) {
    if (x <= 0) return 0;
    if (x > n_seq + 1) return T;
    return min(max(off[x - 1], 0), T);
}

// The rows of one tile slot, and the keys of its sequence (of the other tensor).
struct Slot {
    int first;  // first row of the slot within the sequence
    int base, len;  // the sequence's first row in the packed tensor, and its rows
    int other_base, other_len;  // the same of the tensor on the other side (none outside all sequences)
};

// Whole warp.  Extended sequence x: rows off_at(x) .. off_at(x + 1), x = 0 and n_seq + 1 being the
// rows before and after all sequences.  A search over 31 probes a step; the last step's probes
// already hold the answer, so up to 30 sequences take one round trip to memory, up to 960 two.
__device__ __forceinline__ Slot find_slot(const int32_t *off, const int32_t *other, int n_seq, int T, int T_other,
                                          const Divisor &R, int slot) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seq + 2;
    while (true) {
        const int step = (n + 30) / 31;
        const int x = lo + lane * step;
        const int e = off_at(off, n_seq, T, x);
        int f = 0;
        if (step == 1 && x > 0) f = off == other ? min(e, T_other) : off_at(other, n_seq, T_other, x);
        const bool before = lane * step < n && quotient(e, R) + x <= slot;
        const unsigned m = __ballot_sync(0xffffffffu, before);
        const int p = m ? 31 - __clz(m) : 0;  // at most 30
        if (step == 1) {
            Slot r;
            lo += p;
            r.base = __shfl_sync(0xffffffffu, e, p);
            r.len = max(0, __shfl_sync(0xffffffffu, e, p + 1) - r.base);
            const int ahead = slot - (quotient(r.base, R) + lo);
            r.first = ahead > quotient(r.len, R) ? r.len : ahead * R.d;  // slots past a sequence's rows are empty
            const int a = __shfl_sync(0xffffffffu, f, p), b = __shfl_sync(0xffffffffu, f, p + 1);
            const bool real = lo >= 1 && lo <= n_seq;
            r.other_base = real ? a : 0;
            r.other_len = real ? max(0, b - a) : 0;
            return r;
        }
        lo += p * step;
        n = min(step, n - p * step);
    }
}

inline long long slots_for(long long T, long long R, long long n_seq) { return T / R + n_seq + 2; }

// Polls of a wait before the block gives up.  Every wait here is for work of the same block: where a kernel overlaps
// the one before it, each warp passes wait_for_primary(), which is not counted, before it first polls for anything
// that comes from there.
constexpr int kAttnWaitLimit = 1 << 21;

// A whole warp's wait: all of its lanes go on, or none (tensor memory is moved by warps).  Written to
// be small: the kernels' loops have to stay in the instruction cache.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, unsigned parity, volatile int *abort) {
    int left = kAttnWaitLimit;
#pragma unroll 1
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
        if (__any_sync(0xffffffffu, *abort || --left == 0)) {
            *abort = 1;
            atomicOr(&g_device_fault, 1u);
            return false;
        }
    }
    return true;
}

// The warp's index as a value that the compiler knows to be the same in all lanes.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

// Registers of a block's warpgroups: `GROUPS` that compute and one that loads and issues.  A launch gives
// each thread LAUNCH; the last warpgroup's give theirs up to LESS and the others take MORE.
template <int GROUPS, int LAUNCH, int MORE, int LESS> struct Registers {
    static constexpr int kMore = MORE, kLess = LESS;
    static_assert(GROUPS * MORE + LESS <= (GROUPS + 1) * LAUNCH, "a warpgroup would wait for registers for good");
};

// D = A B^T over DP channels, `dim` of them in use, A and B K-major tiles whose column panels are `a_panel` and
// `b_panel` bytes.
template <int DP, int A_PANEL, int B_PANEL>
__device__ __forceinline__ void mma_channels(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int dim) {
    constexpr int N = Tile<DP>::kCols / 16;  // steps in a panel
    mma_ss_one<N, 2, 2>(d, a, b, idesc, false);
    if constexpr (Tile<DP>::kPanels == 2) {
        if (dim <= 96) mma_ss_one<2, 2, 2>(d, a + A_PANEL / 16, b + B_PANEL / 16, idesc, true);
        else mma_ss_one<N, 2, 2>(d, a + A_PANEL / 16, b + B_PANEL / 16, idesc, true);
    }
}

// Bits lo .. hi - 1 of a word.
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 32);
    return hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
}

// Zeroes rows [from, to) of a swizzled tile by the first `threads` threads of a block or a warp's
// lanes (32); whole rows, so the swizzle does not matter.
template <int DP>
__device__ __forceinline__ void zero_rows(uint32_t tile, int rows_in_panel, int from, int to, int threads) {
    constexpr int CH = Tile<DP>::kRowBytes / 16;
    const int n = (to - from) * CH;
#pragma unroll 1
    for (int p = 0; p < Tile<DP>::kPanels; ++p) {
        const uint32_t a = tile + p * rows_in_panel * Tile<DP>::kRowBytes + from * Tile<DP>::kRowBytes;
#pragma unroll 1
        for (int i = threadIdx.x & (threads - 1); i < n; i += threads)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a + i * 16), "r"(0) : "memory");
    }
}

// Bytes that a box of `rows` tile rows brings (boxes past a tensor's end are filled up with zeros).
template <int DP> __device__ __forceinline__ unsigned box_bytes(int rows) {
    return rows * Tile<DP>::kRowBytes * Tile<DP>::kPanels;
}

// ---------------------------------------------------------------------------------------------
// Forward.
//
// A row tile is 128 rows (queries x packed heads) of one sequence and key head; keys come in tiles.
// Per key tile S = Q K^T (both operands in shared memory) into TMEM; a warpgroup turns it into
// P = exp2(scale log2(e) (S - m)) in registers, one row per thread, and writes it back as bf16 over
// S; O += P V takes P from TMEM.  The reference m of a row is its running maximum, but moves only
// when that grew by more than kLazy (in powers of two; P and its sum stay below 2^kLazy times their
// true scale, far from any limit in float32, and bf16's relative rounding does not depend on the
// scale), so that O in TMEM is seldom rescaled.  P is rounded to bf16 because that is what the
// tensor core takes; its row sum is kept in float32 from the unrounded values.  The last tile of
// the keys works on as many columns as are seen, in steps of 16, and warps whose rows are all past
// the sequence do none of it.
// ---------------------------------------------------------------------------------------------
constexpr float kLazy = 8.0f;

// The largest of N values.
template <int N> __device__ __forceinline__ float max_of(const float *s) {
    float a[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) a[c] = fmaxf(s[c], s[c + 4]);
#pragma unroll
    for (int c = 8; c < N; c += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaxf(fmaxf(a[e], s[c + e]), s[c + e + 4]);
    }
    return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
}

// A row's softmax so far: P and sum are relative to exp2(m scale log2(e)).  A tile's row that is no query of its
// sequence holds whatever lies behind those (another sequence's, or what shared memory held before): it starts from
// m = inf, where no score moves the reference, and so does not change how the other rows' weights round.
struct RowState {
    float m, sum;
    __device__ explicit RowState(bool live) : m(live ? -INFINITY : INFINITY), sum(0.0f) {}
};

// 2^(sc s + ref) of N values in pairs, packed to bf16; adds them to acc[2].  With POLY one pair of eight takes
// the FMA pipe: 8192 + 3001 + 130 causal tokens, 8 / 2 heads of 128, forward, 156 us without, 152 with one, 151
// with two of eight (three: slower again).  The short kernel, whose four blocks hide more, gains nothing by it.
template <int N, bool POLY>
__device__ __forceinline__ void exp_pack(const float *s, float sc, float ref, uint32_t *p, float2 *acc) {
    const float2 sc2 = make_float2(sc, sc), ref2 = make_float2(ref, ref);
#pragma unroll
    for (int c = 0; c < N / 2; ++c) {
        float2 x = fma2(make_float2(s[2 * c], s[2 * c + 1]), sc2, ref2);
        if (POLY && (c % 8 == 4)) {
            x = exp2_poly(x);
        } else {
            x.x = exp2_fast(x.x);
            x.y = exp2_fast(x.y);
        }
        acc[c & 1] = add2(acc[c & 1], x);
        p[c] = pack_bf16(x.x, x.y);
    }
}

// Whole warp: moves the reference to the new maximum where some live row's grew far enough, and O and the
// sum with it.
template <int DP> __device__ __forceinline__ void move_reference(RowState &r, uint32_t to, float mx, bool first,
                                                                 float sc) {
    if (first) {
        r.m = fmaxf(r.m, mx);
    } else if (__any_sync(0xffffffffu, mx * sc > r.m * sc + kLazy)) {
        const float to_m = fmaxf(r.m, mx);
        const float f = to_m == -INFINITY ? 1.0f : exp2_fast((r.m - to_m) * sc);
        r.m = to_m;
        r.sum *= f;
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
            float o[16];
            tmem_ld16(to + c, o);
            tmem_wait_ld();
            pin<16>(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= f;
            tmem_st16(to + c, reinterpret_cast<uint32_t *>(o));
        }
    }
}

// Whole warp: one key tile of S at TMEM `ts` (this warp's lanes) becomes P at `tp`; `to` is O.  `cols`
// columns are in use, of which this row sees `seen`; `all` says that every row sees all KEYS.
// loaded() is called once S has been read, settle() before P is written or O touched (it returns
// false to give up), written(half) after each half of P.
// Tiles that are seen whole, the many, are read once into registers and run straight through; the
// others go over S twice in a small loop.
template <int DP, typename Loaded, typename Settle, typename Written>
__device__ __forceinline__ bool softmax_tile(RowState &r, uint32_t ts, uint32_t tp, uint32_t to, int cols, bool all,
                                             int seen, bool first, float sc, Loaded loaded, Settle settle,
                                             Written written) {
    constexpr int KEYS = 128;
    float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    if (all) {
        float s[KEYS];
#pragma unroll
        for (int c = 0; c < KEYS; c += 32) tmem_ld32(ts + c, s + c);
        tmem_wait_ld();
        pin<KEYS>(s);
        loaded();
        const float mx = max_of<KEYS>(s);
        if (!settle()) return false;
        move_reference<DP>(r, to, mx, first, sc);
        const float ref = r.m == -INFINITY ? 0.0f : -r.m * sc;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t p[KEYS / 4];
            exp_pack<KEYS / 2, true>(s + h * (KEYS / 2), sc, ref, p, acc);
            tmem_st32(tp + h * 32, p);
            tmem_wait_st();
            written(h);
        }
    } else {
        float mx = -INFINITY;
        float s[32];
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
            tmem_ld32(ts + c, s);
            tmem_wait_ld();
            pin<32>(s);
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = c + e < seen ? fmaxf(mx, s[e]) : mx;
        }
        if (!settle()) return false;
        move_reference<DP>(r, to, mx, first, sc);
        const float ref = r.m == -INFINITY ? 0.0f : -r.m * sc;
        // P of 32 keys takes 16 columns: over S it stays behind what has been read.
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
            tmem_ld32(ts + c, s);
            tmem_wait_ld();
            pin<32>(s);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = c + e < seen ? s[e] : -INFINITY;
            uint32_t p[16];
            exp_pack<32, false>(s, sc, ref, p, acc);
            tmem_st16(tp + c / 2, p);
        }
        tmem_wait_st();
        loaded();
        written(0);
        written(1);
    }
    r.sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
    return true;
}

// The same for one warpgroup's tile of 64 keys, P over S.  Masked tiles run straight through too: in short
// sequences they are many.
template <int DP>
__device__ __forceinline__ void softmax_tile64(RowState &r, uint32_t ts, uint32_t to, int cols, bool all, int seen,
                                               bool first, float sc) {
    float s[64];
    tmem_ld32(ts, s);
    if (cols > 32) tmem_ld32(ts + 32, s + 32);
    tmem_wait_ld();
    pin<64>(s);
    if (!all) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t m = bits(0, seen - h * 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) s[h * 32 + c] = m & (1u << c) ? s[h * 32 + c] : -INFINITY;
        }
    }
    move_reference<DP>(r, to, max_of<64>(s), first, sc);
    const float ref = r.m == -INFINITY ? 0.0f : -r.m * sc;
    float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    uint32_t p[32];
    if (all) {
        exp_pack<64, false>(s, sc, ref, p, acc);
        tmem_st32(ts, p);
    } else {
        exp_pack<32, false>(s, sc, ref, p, acc);
        tmem_st16(ts, p);
        if (cols > 32) {
            exp_pack<32, false>(s + 32, sc, ref, p + 16, acc);
            tmem_st16(ts + 16, p + 16);
        }
    }
    tmem_wait_st();
    r.sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
}

// Where results go.  `low` is what a result lost in its rounding to bf16, itself in bf16, for the backward
// pass: delta = o.g taken from the rounded o alone is off by as much as dS's own rounding in short sequences.
struct FwdOut {
    bf16 *out, *low;         // low, lse: or null
    float *lse;
    float *part, *part_lse;  // of shared-out keys, by block: [blocks][part_rows][D] and [blocks][part_rows]
    int part_rows;
};

// Eight values of a result and, where that is wanted, what their rounding lost.
__device__ __forceinline__ void store_result(const FwdOut &f, size_t at, const float *v) {
    store_vec<bf16, 8>(f.out + at, v);
    if (f.low) {
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = v[e] - to_f32(from_f32<bf16>(v[e]));
        store_vec<bf16, 8>(f.low + at, rest);
    }
}

// Whole warp: a row's result from O (or zeros) and its log-sum-exp.  With PAIR columns `from` .. `end` of a row's sum
// of two, O times `times` and `other` (the first column's place) times `more`; where `part_row` is not negative,
// to that row of the parts.
template <int DP, bool PAIR>
__device__ __forceinline__ void write_row(const AttnArgs &A, const FwdOut &f, long long part_row, const RowState &r,
                                          uint32_t to, bool any, bool live, size_t token, int head, int from = 0,
                                          int end = DP, float times = 1.0f, const float *other = nullptr,
                                          float more = 0.0f) {
    const float inv = r.sum == 0.0f ? 0.0f : 1.0f / r.sum;
    const bool is_part = PAIR && part_row >= 0;
    if (live && from == 0) {
        const float l = r.sum == 0.0f ? -INFINITY : r.m * A.scale + logf(r.sum);
        if (is_part) f.part_lse[part_row] = l;
        else if (f.lse) f.lse[(size_t)head * A.Tq + token] = l;
    }
    const size_t at = (is_part ? (size_t)part_row : token * A.Hq + head) * A.D;
#pragma unroll 1
    for (int c = PAIR ? from : 0; c < (PAIR ? end : DP); c += 16) {
        float o[16];
        if (any) {
            tmem_ld16(to + c, o);
            tmem_wait_ld();
            pin<16>(o);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.0f;
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            if (c + e >= A.D) continue;
            float x[8];
            if (PAIR) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 y = *reinterpret_cast<const float4 *>(other + (c - from) + e + i);
                    x[i] = fmaf(y.x, more, o[e + i] * times) * inv;
                    x[i + 1] = fmaf(y.y, more, o[e + i + 1] * times) * inv;
                    x[i + 2] = fmaf(y.z, more, o[e + i + 2] * times) * inv;
                    x[i + 3] = fmaf(y.w, more, o[e + i + 3] * times) * inv;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = o[e + i] * inv;
            }
            if (is_part) store_vec<float, 8>(f.part + at + c + e, x);
            else store_result(f, at + c + e, x);
        }
    }
}

// Columns of a key tile that a row tile works on.
__device__ __forceinline__ int tile_cols(int sees, int k0, int keys) { return min(keys, (sees - k0 + 15) & ~15); }

// ---- long sequences: two row tiles to a block, roles by warp -------------------------------------
// One warp loads, one issues the matrix products, a warpgroup serves each row tile: while the
// tensor core works on one tile, the other's exponentials run, and K and V are read from L2 once
// for 256 rows.  128 keys a tile.  The warpgroups take their registers from the other two warps
// (setmaxnreg): a row of S is 128 values.
// What bounds it is the chain of a row tile from S through the maximum, the exponentials and P to P V, of
// which two tiles in flight hide about half: 10,052 causal tokens of six prompts, 16 / 4 heads of 128, take
// 122 us, 1020 TFLOP/s of the products that the mask leaves (62% of the measured peak), with the tensor pipe
// 50%, the special-function unit 45% and the issue slots 37% busy.  Four warpgroups, two to a row tile, took
// 150 us: what each waits for is the other roles, not its own work.
// Where the launch has no more row tiles than SMs, two to a block would leave SMs without one: a block has one, and
// its two halves take the key tiles in turn, each with sums of its own, which they add at the end through
// shared memory (ALT).  With few row tiles their keys are also shared out over blocks (SPLIT): each writes its
// normalised part in float32 and its lse, and attn_join_kernel adds them by weight.
template <int DP, bool ALT> struct LongShape {
    static constexpr int kKeys = 128;
    static constexpr int kTileBytes = 128 * DP * 2;
    static constexpr int kStages = 4;
    static constexpr int kThreads = 384;
    using Regs = Registers<2, 168, 208, 88>;  // 65536 / 384 -> 168
    static constexpr int kTmem = 512;
    static constexpr size_t kSmem = 1024 + (size_t)(2 + kStages) * kTileBytes;
    static constexpr int kLeast = 8;  // key tiles to a block where they are shared out
    static_assert(!ALT || 128 * (DP + 8) * 4 <= kStages * kTileBytes, "the halves' sums");
    // TMEM: S of both tiles (2 x 128), O of both (2 x DP), and P (2 x 64) where there is room for it;
    // with 128 channels there is none and P lies over S.  P of its own lets the next S be formed while
    // this one's exponentials run.
    static constexpr bool kOwnP = DP <= 64 && !ALT;
    static constexpr int kO = 256, kP = kOwnP ? 256 + 2 * DP : 0, kPStep = kOwnP ? 64 : 128;
};
struct LongShared {
    uint64_t q_full[2], kv_full[4], kv_raw, kv_empty[4], s_full[2], s_free[2], p_half[2][2], o_done[2], drain;
    uint32_t tmem;
    int abort;
    long long part_row;  // of the block's first row among the parts; negative: its results are whole
};

struct LongRange {
    int sees[2];    // keys that each row tile works on
    int cnt[2];     // key tiles that each row tile (or, ALT, each half of the block) works on
    int j0, end;    // key tiles of the block
    int tok[2];     // tokens of each row tile
};

// Shared-out keys.  The host does not know the lengths, so each block looks at all of them: a slot with w key
// tiles gets ceil(w / c) blocks a head, with the smallest c that the launch's blocks allow.  Eight single tokens
// over 1 to 16384 keys, 16 / 4 heads of 128, take 39.3 us, of them 3.5 until a block has its share, 26 for
// its keys (5.9 TB/s all together), 7 for the join; with four blocks to each slot, whatever its length, 48.
constexpr int kSharedSlots = 384;  // at most, so that a thread sees to each

struct SharedOut {
    int off[kSharedSlots + 3], other[kSharedSlots + 3];  // rows and keys at which the extended sequences begin
    int tiles[kSharedSlots];                             // of each slot; 0 only where it has no rows
};

// As find_slot, from the copy of the offsets, by one thread.
__device__ __forceinline__ Slot shared_slot(const AttnArgs &A, const SharedOut &so, int slot) {
    int lo = 0, n = A.n_seq + 2;  // the last x among lo .. lo + n - 1 that begins at or before the slot
#pragma unroll 1
    while (n > 1) {
        const int half = n >> 1;
        const bool before = quotient(so.off[lo + half], A.slot_rows) + lo + half <= slot;
        lo += before ? half : 0;
        n = before ? n - half : half;
    }
    Slot r;
    r.base = so.off[lo];
    r.len = max(0, so.off[lo + 1] - r.base);
    const int ahead = slot - (quotient(r.base, A.slot_rows) + lo);
    r.first = ahead > quotient(r.len, A.slot_rows) ? r.len : ahead * A.slot_rows.d;
    const bool real = lo >= 1 && lo <= A.n_seq;
    r.other_base = real ? so.other[lo] : 0;
    r.other_len = real ? max(0, so.other[lo + 1] - r.other_base) : 0;
    return r;
}

// All threads of a block (two barriers).
__device__ __forceinline__ void count_tiles(const AttnArgs &A, SharedOut &so, int slots) {
#pragma unroll 1
    for (int x = threadIdx.x; x < A.n_seq + 3; x += blockDim.x) {
        so.off[x] = off_at(A.q_off, A.n_seq, A.Tq, x);
        so.other[x] = off_at(A.k_off, A.n_seq, A.Tk, x);
    }
    __syncthreads();
#pragma unroll 1
    for (int x = threadIdx.x; x < slots; x += blockDim.x) {
        const Slot q = shared_slot(A, so, x);
        const int end = min(q.len, q.first + A.slot_rows.d);
        const int sees = A.causal ? min(q.other_len, max(0, end + q.other_len - q.len)) : q.other_len;
        so.tiles[x] = q.first >= q.len ? 0 : max(1, (sees + 127) / 128);
    }
    __syncthreads();
}

// Whole warp: the smallest c, and `least` at least, with which a launch of `blocks` suffices: sum ceil(w / c) of all
// slots and heads.  There are at least as many blocks as slots times heads.
__device__ __forceinline__ unsigned share_size(const AttnArgs &A, const SharedOut &so, int slots, unsigned least,
                                               unsigned blocks) {
    const unsigned lane = threadIdx.x & 31, heads = A.heads.d;
    unsigned total = 0, live = 0, most = 0;  // total: at most 384 slots of 2^23 tiles
#pragma unroll 1
    for (int x = lane; x < slots; x += 32) {
        const unsigned w = so.tiles[x];
        total += w;
        live += w > 0;
        most = max(most, w);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    live = __reduce_add_sync(0xffffffffu, live);
    most = __reduce_max_sync(0xffffffffu, most);
    const unsigned long long all = (unsigned long long)total * heads;
    auto over = [&](unsigned n) {  // all / n, rounded up
        if (all >> 31) return (unsigned)min((all + n - 1) / n, 0x7fffffffull);
        return ((unsigned)all + n - 1) / n;
    };
    const unsigned spare = blocks - live * heads;
    unsigned lo = max(least, over(blocks));
    unsigned hi = max(lo, most);  // a block to each; and as ceil(w / c) < w / c + 1:
    if (spare > 0) hi = min(hi, max(lo, over(spare)));
#pragma unroll 1
    while (lo < hi) {
        const unsigned c = (lo + hi) / 2;
        unsigned n = 0;
#pragma unroll 1
        for (int x = lane; x < slots; x += 32) n += (so.tiles[x] + c - 1) / c;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n * heads <= blocks) hi = c;
        else lo = c + 1;
    }
    return lo;
}

struct Share {
    int slot, head;    // slot -1: nothing left for this block
    int which, parts;  // of the slot's key tiles
};

// Whole warp: block b's share, c key tiles at most.
__device__ __forceinline__ Share find_share(const AttnArgs &A, const SharedOut &so, int slots, unsigned c, int b) {
    const int lane = threadIdx.x & 31, heads = A.heads.d;
    int before = 0;
#pragma unroll 1
    for (int x0 = 0; x0 < slots; x0 += 32) {
        const int parts = x0 + lane < slots ? (so.tiles[x0 + lane] + c - 1) / c : 0;
        int upto = parts * heads;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        upto += before;
        const unsigned m = __ballot_sync(0xffffffffu, upto > b);
        if (m) {
            const int p = __ffs(m) - 1;
            Share r;
            r.slot = x0 + p;
            r.parts = __shfl_sync(0xffffffffu, parts, p);
            const int rest = b - (__shfl_sync(0xffffffffu, upto, p) - r.parts * heads);
            r.which = quotient(rest, A.heads);
            r.head = rest - r.which * heads;
            return r;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
    }
    return {-1, 0, 0, 0};
}

// Whole warp; returns how many tiles of K and V were asked for.
template <int DP, bool ALT>
__device__ int long_load(const AttnArgs &A, const CUtensorMap *mq, const CUtensorMap *mk, const CUtensorMap *mv,
                         LongShared &sh, uint32_t smem_q, uint32_t smem_kv, const LongRange &r, int kvh, int qhead,
                         int qrow, int tok_per_tile, int krow, int klen) {
    using S = LongShape<DP, ALT>;
    using TL = Tile<DP>;
    volatile int *abort = &sh.abort;
    const int loads = 2 * (r.end - r.j0);
    int issued = 0;
    unsigned raw_phase = 0;
#pragma unroll 1
    for (; issued < loads; ++issued) {
        const int st = issued % S::kStages;
        if (issued >= S::kStages && !wait_warp(&sh.kv_empty[st], ((issued / S::kStages) - 1) & 1, abort)) break;
        const int j = r.j0 + (issued >> 1);
        const bool is_v = issued & 1;
        // The last tile of V may reach into rows that are not this sequence's: P is 0 there, but
        // 0 x inf is not, so they are cleared before the tensor core sees the tile.
        const int foreign = is_v ? (j + 1) * S::kKeys - klen : 0;
        const uint32_t dst = smem_kv + st * S::kTileBytes;
        uint64_t *bar = foreign > 0 ? &sh.kv_raw : &sh.kv_full[st];
        mbar_arrive_expect_one(bar, S::kTileBytes);
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p)
            tma_load_3d_one(dst + p * 128 * TL::kRowBytes, is_v ? mv : mk, bar, p * TL::kCols, kvh,
                            krow + j * S::kKeys);
        if (issued == 0) {
#pragma unroll
            for (int t = 0; t < (ALT ? 1 : 2); ++t) {
                if (r.cnt[t] == 0) continue;
                mbar_arrive_expect_one(&sh.q_full[t], box_bytes<DP>(tok_per_tile * A.pack));
#pragma unroll
                for (int p = 0; p < TL::kPanels; ++p)
                    tma_load_3d_one(smem_q + t * S::kTileBytes + p * 128 * TL::kRowBytes, mq, &sh.q_full[t],
                                    p * TL::kCols, qhead, qrow + t * tok_per_tile);
            }
        }
        if (foreign > 0) {
            if (!wait_warp(&sh.kv_raw, raw_phase, abort)) {
                mbar_drain(&sh.kv_raw, raw_phase, kAttnWaitLimit);
                break;
            }
            raw_phase ^= 1;
            zero_rows<DP>(dst, 128, S::kKeys - foreign, S::kKeys, 32);
            fence_async_smem();
            __syncwarp();
            mbar_arrive_one(&sh.kv_full[st]);
        }
    }
    return issued;
}

// After a wait gave up: every copy of this block that may still be landing.
template <int DP, bool ALT> __device__ void long_drain(LongShared &sh, const LongRange &r, int issued) {
    using S = LongShape<DP, ALT>;
    for (int t = 0; t < (ALT ? 1 : 2); ++t)
        if (r.cnt[t] > 0) mbar_drain(&sh.q_full[t], 0, kAttnWaitLimit);
    for (int i = max(0, issued - S::kStages); i < issued; ++i)
        mbar_drain(&sh.kv_full[i % S::kStages], (i / S::kStages) & 1, kAttnWaitLimit);
}

// Whole warp.
template <int DP, bool ALT>
__device__ bool long_mma_loop(LongShared &sh, uint32_t smem_q, uint32_t smem_kv, const LongRange &r, uint32_t tmem,
                              int dim) {
    using S = LongShape<DP, ALT>;
    using TL = Tile<DP>;
    const uint32_t id_o = mma_idesc(128, (dim + 15) & ~15, true);
    constexpr uint32_t kSbo = 8 * TL::kRowBytes, kLbo = 128 * TL::kRowBytes;
    volatile int *abort = &sh.abort;
    const uint64_t q_desc = smem_desc<TL::kRowBytes>(smem_q, 16, kSbo);
    const uint64_t k_desc = smem_desc<TL::kRowBytes>(smem_kv, 16, kSbo);
    const uint64_t v_desc = smem_desc<TL::kRowBytes>(smem_kv, kLbo, kSbo);
    auto scores = [&](int t, int st, int j) {
        const uint32_t id = mma_idesc(128, tile_cols(r.sees[t], j * S::kKeys, S::kKeys), false);
        const uint64_t a = q_desc + (ALT ? 0 : t) * (S::kTileBytes / 16), b = k_desc + st * (S::kTileBytes / 16);
        mma_channels<DP, kLbo, kLbo>(tmem + t * 128, a, b, id, dim);
        tc_commit_one(&sh.s_full[t]);
    };
    auto kv = [&](int load) {  // waits for a load of the ring; returns its stage or -1
        return wait_warp(&sh.kv_full[load % S::kStages], (load / S::kStages) & 1, abort) ? load % S::kStages : -1;
    };
    // The key tile of a row tile's i-th round; its loads are the ring's 2 (j - j0) for K and the next for V.
    auto tile = [&](int t, int i) { return r.j0 + (ALT ? 2 * i + t : i); };
    int st = -1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (r.cnt[t] == 0) continue;
        if (ALT || st < 0)
            if ((st = kv(2 * (tile(t, 0) - r.j0))) < 0) return false;
        if (!wait_warp(&sh.q_full[ALT ? 0 : t], 0, abort)) return false;
        tc_fence_after();
        scores(t, st, tile(t, 0));
        if (ALT) tc_commit_one(&sh.kv_empty[st]);
    }
    if (!ALT) tc_commit_one(&sh.kv_empty[st]);
    // O_t += P V of tile i, each half as soon as it is written.
    auto product = [&](int t, int i, int sv) {
        const int steps = tile_cols(r.sees[t], tile(t, i) * S::kKeys, S::kKeys) / 16;
        const uint64_t b = v_desc + sv * (S::kTileBytes / 16);
        const uint32_t o = tmem + S::kO + t * DP, p = tmem + S::kP + t * S::kPStep;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!wait_warp(&sh.p_half[t][h], i & 1, abort)) return false;
            tc_fence_after();
            if (steps == 8) {
                mma_ts_one<4, TL::kRowBytes>(o, p + h * 32, b + h * 4 * TL::kRowBytes, id_o, i > 0 || h > 0);
            } else {
#pragma unroll 1
                for (int k = h * 4; k < min(steps, h * 4 + 4); ++k)
                    mma_ts_one<1, 0>(o, p + k * 8, b + k * TL::kRowBytes, id_o, i > 0 || k > 0);
            }
        }
        tc_commit_one(&sh.o_done[t]);
        return true;
    };
    const int n = max(r.cnt[0], r.cnt[1]);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        int sv = -1, sk = -1;
        if (S::kOwnP) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (r.cnt[t] - i <= 1) continue;
                if (sk < 0 && (sk = kv(2 * i + 2)) < 0) return false;
                if (!wait_warp(&sh.s_free[t], i & 1, abort)) return false;
                tc_fence_after();
                scores(t, sk, tile(t, i + 1));
            }
            if (sk >= 0) tc_commit_one(&sh.kv_empty[sk]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int left = r.cnt[t] - i;  // key tiles of this row tile from here on
            if (left > 0) {
                if (ALT || sv < 0)
                    if ((sv = kv(2 * (tile(t, i) - r.j0) + 1)) < 0) return false;
                if (!product(t, i, sv)) return false;
                if (ALT) tc_commit_one(&sh.kv_empty[sv]);
            }
            if (!S::kOwnP && left > 1) {
                if (ALT || sk < 0)
                    if ((sk = kv(2 * (tile(t, i + 1) - r.j0))) < 0) return false;
                tc_fence_after();
                scores(t, sk, tile(t, i + 1));
                if (ALT) tc_commit_one(&sh.kv_empty[sk]);
            }
        }
        if (!ALT && sv >= 0) tc_commit_one(&sh.kv_empty[sv]);
        if (!ALT && !S::kOwnP && sk >= 0) tc_commit_one(&sh.kv_empty[sk]);
    }
    return true;
}

// The two halves of an ALT block's warpgroups.
__device__ __forceinline__ void half_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int DP, bool ALT, bool SPLIT>
__global__ void __launch_bounds__(LongShape<DP, ALT>::kThreads, 1)
attn_forward_long_kernel(const AttnArgs A, const __grid_constant__ CUtensorMap mq,
                         const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                         const FwdOut f, int slots) {
    static_assert(ALT || !SPLIT, "keys are shared out by single row tiles");
    using S = LongShape<DP, ALT>;
    extern __shared__ unsigned char dyn[];
    __shared__ LongShared sh;
    const int warp = warp_index();
    const int per = 128 / A.pack;  // tokens in a row tile
    auto start = [&] {
        if (warp != 8) return;
        if ((threadIdx.x & 31) == 0) {
            for (int t = 0; t < 2; ++t) {
                mbar_init(&sh.q_full[t], 1);
                mbar_init(&sh.s_full[t], 1);
                mbar_init(&sh.s_free[t], 4);
                mbar_init(&sh.p_half[t][0], 4);
                mbar_init(&sh.p_half[t][1], 4);
                mbar_init(&sh.o_done[t], 1);
            }
            for (int i = 0; i < S::kStages; ++i) {
                mbar_init(&sh.kv_full[i], 1);
                mbar_init(&sh.kv_empty[i], 1);
            }
            mbar_init(&sh.kv_raw, 1);
            mbar_init(&sh.drain, 1);
            sh.abort = 0;
            mbar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&sh.tmem, S::kTmem);
    };
    int slot, hx;
    Slot q;
    Share share{0, 0, 0, 1};
    if constexpr (SPLIT) {
        __shared__ SharedOut so;
        launch_dependents();
        start();
        tc_fence_before();
        count_tiles(A, so, slots);
        tc_fence_after();
        share = find_share(A, so, slots, share_size(A, so, slots, S::kLeast, gridDim.x), blockIdx.x);
        if (share.slot < 0) {
            if (warp == 8) tmem_dealloc(sh.tmem, S::kTmem);
            return;
        }
        slot = share.slot;
        hx = share.head;
        q = shared_slot(A, so, slot);
    } else {
        const int s = quotient(blockIdx.x, A.heads);
        hx = blockIdx.x - s * A.heads.d;
        // Later slots first: under a causal mask they see more keys.
        slot = slots - 1 - s;
        q = find_slot(A.q_off, A.k_off, A.n_seq, A.Tq, A.Tk, A.slot_rows, slot);
    }
    if (!SPLIT && q.first >= q.len) return;
    const int kbase = q.other_base, klen = q.other_len;
    const int kvh = hx / A.subs;
    const int qhead = kvh * (A.Hq / A.Hkv) + (hx % A.subs) * A.pack;

    LongRange r;
    int n[2];  // key tiles of each row tile
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = q.first + (ALT ? 0 : t * per);
        r.tok[t] = min(per, max(0, q.len - first));
        const int last = first + r.tok[t] - 1;
        r.sees[t] = r.tok[t] == 0 ? 0 : A.causal ? min(klen, max(0, last + 1 + klen - q.len)) : klen;
        n[t] = (r.sees[t] + S::kKeys - 1) / S::kKeys;
    }
    r.j0 = 0;
    r.end = max(n[0], n[1]);
    if (SPLIT) {
        const int each = (r.end + share.parts - 1) / share.parts;
        r.j0 = min(r.end, each * share.which);
        r.end = min(r.end, r.j0 + each);
        if (threadIdx.x == 0) {
            sh.part_row = share.parts > 1 ? (long long)blockIdx.x * f.part_rows : -1;
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
        r.cnt[t] = ALT ? (r.end - r.j0 + 1 - t) / 2 : max(0, min(n[t], r.end) - r.j0);

    if (!SPLIT) start();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    const uint32_t smem_q = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t smem_kv = smem_q + 2 * S::kTileBytes;

    int issued = 0;
    if (warp >= 8) {
        regs_less<S::Regs::kLess>();
        if (warp == 8) {
            if (r.end > r.j0) long_mma_loop<DP, ALT>(sh, smem_q, smem_kv, r, tmem, A.D);
        } else if (warp == 9) {
            issued = long_load<DP, ALT>(A, &mq, &mk, &mv, sh, smem_q, smem_kv, r, kvh, qhead, q.base + q.first, per,
                                        kbase, klen);
        }
    } else {
        regs_more<S::Regs::kMore>();
        const int t = warp >> 2;
        if (r.tok[t] > 0) {
            volatile int *abort = &sh.abort;
            const uint32_t lane_base = (uint32_t)(warp & 3) << 21;  // lane 32 (w % 4)
            const uint32_t ts = tmem + lane_base + t * 128, to = tmem + lane_base + S::kO + t * DP;
            const uint32_t tp = tmem + lane_base + S::kP + t * S::kPStep;
            const int row = threadIdx.x & 127;
            const int tok_first = q.first + (ALT ? 0 : t * per), tok = tok_first + row_token(A, row);
            const bool live = row_token(A, row) < r.tok[t];
            const bool warp_live = (row & ~31) < r.tok[t] * A.pack;
            const int limit = A.causal ? min(klen, max(0, tok + 1 + klen - q.len)) : klen;
            // Keys that every row of the tile sees (rows past the last token do not count).
            const int all_see = A.causal ? min(klen, tok_first + 1 + klen - q.len) : klen;
            RowState rs(live);
            const int n = r.cnt[t];
            bool ok = true;
#pragma unroll 1
            for (int i = 0; i < n && ok; ++i) {
                ok = wait_warp(&sh.s_full[t], i & 1, abort);
                if (!ok) break;
                tc_fence_after();
                const int k0 = (r.j0 + (ALT ? 2 * i + t : i)) * S::kKeys;
                auto loaded = [&] {
                    if (!S::kOwnP) return;
                    tc_fence_before();
                    mbar_arrive_one(&sh.s_free[t]);
                };
                // P V of the tile before: done with S of this one where P lies over S (issue order).
                auto settle = [&] {
                    if (!S::kOwnP || i == 0) return true;
                    if (!wait_warp(&sh.o_done[t], (i - 1) & 1, abort)) return false;
                    tc_fence_after();
                    return true;
                };
                auto written = [&](int h) {
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_one(&sh.p_half[t][h]);
                };
                if (warp_live) {
                    ok = softmax_tile<DP>(rs, ts, tp, to, tile_cols(r.sees[t], k0, S::kKeys),
                                          k0 + S::kKeys <= all_see, limit - k0, i == 0, A.scale_log2, loaded, settle,
                                          written);
                } else {
                    loaded();
                    ok = settle();
                    written(0);
                    written(1);
                }
            }
            if (ok && n > 0) ok = wait_warp(&sh.o_done[t], (n - 1) & 1, abort);
            tc_fence_after();
            const size_t token = (size_t)q.base + tok;
            const int head = qhead + row_head(A, row);
            const long long part_row = SPLIT && sh.part_row >= 0 ? sh.part_row + row : -1;
            if (!ALT) {
                if (ok) write_row<DP, false>(A, f, -1, rs, to, n > 0, live, token, head);
            } else {
                // Each half gives the other its sums of half of the channels, through the room of K and V once
                // both are through with it.
                constexpr int kSide = DP / 2 + 4;  // four more: its maximum and sum, and other banks for each row
                float *side = reinterpret_cast<float *>(dyn + (smem_kv - smem_u32(dyn))) + row * kSide;
                float *give = side + (1 - t) * 128 * kSide, *take = side + t * 128 * kSide;
                half_barrier();
                if (ok && warp_live) {
                    if (live) *reinterpret_cast<float2 *>(give + DP / 2) = make_float2(rs.m, rs.sum);
#pragma unroll 1
                    for (int c = 0; c < DP / 2; c += 16) {
                        float o[16];
                        if (n > 0) {
                            tmem_ld16(to + (1 - t) * (DP / 2) + c, o);
                            tmem_wait_ld();
                            pin<16>(o);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = 0.0f;
                        }
                        if (!live) continue;
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<float4 *>(give + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                half_barrier();
                if (__all_sync(0xffffffffu, ok && !*abort) && warp_live) {
                    float a = 0.0f, b = 0.0f;
                    if (live) {
                        const float2 y = *reinterpret_cast<const float2 *>(take + DP / 2);
                        const float m = fmaxf(rs.m, y.x);
                        a = rs.m == -INFINITY ? 0.0f : exp2f((rs.m - m) * A.scale_log2);
                        b = y.x == -INFINITY ? 0.0f : exp2f((y.x - m) * A.scale_log2);
                        // In the same order in both, for the same bits.
                        const float s0 = t == 0 ? rs.sum * a : y.y * b, s1 = t == 0 ? y.y * b : rs.sum * a;
                        rs.m = m;
                        rs.sum = s0 + s1;
                    }
                    write_row<DP, true>(A, f, part_row, rs, to, n > 0, live, token, head, t * (DP / 2),
                                               (t + 1) * (DP / 2), a, take, b);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (sh.abort && warp == 9 && (threadIdx.x & 31) == 0) long_drain<DP, ALT>(sh, r, issued);
    if (warp == 8) {
        if (sh.abort) {
            tc_commit_one(&sh.drain);
            mbar_drain(&sh.drain, 0, kAttnWaitLimit);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmem);
    }
}

// ---- short sequences: one row tile at a time, several blocks to an SM ----------------------------
// With a few key tiles to a row tile, most of a block's time would be its start and its end; four blocks
// to an SM (two with 128 channels) cover each other's instead of roles within one, and stay for the whole
// launch: each takes every gridDim.x-th row tile, and looks up and asks for the next one's Q, K and V while
// it works (104 x 300 tokens of 8 heads of 32: blocks that come and go cost 13.7 us by themselves, and
// finding their rows 14 more, of 62).  128 threads: each owns a row, warp 0 also issues the copies and
// the products.  64 keys a tile, so that S and O of four blocks fit TMEM and a row of S is 64 registers.
// Those 104 x 300 tokens take 57 us (62 with `low`), 32 x 145 of 6 heads of 64 12.0 us: latencies still (40% of the
// special functions' rate, 41% of the issue slots); 256 threads, half a row each, took 66 and 15.3 us.
template <int DP> struct ShortShape {
    static constexpr int kKeys = 64;
    static constexpr int kQBytes = 128 * DP * 2;
    static constexpr int kTileBytes = kKeys * DP * 2;
    static constexpr int kTmem = DP <= 64 ? 128 : 256;  // S 64, O DP
    static constexpr int kBlocks = DP <= 64 ? 4 : 2;
    static constexpr size_t kSmem = 1024 + kQBytes + 4 * (size_t)kTileBytes;
};

struct ShortShared {
    uint64_t k_full[2], v_full[2], s_full, o_done, drain;
    uint32_t tmem;
    int abort;
};

// One row tile's work.
struct ShortItem {
    int qrow, qhead, tok0;   // first packed row, first head, first token within the sequence
    int ntok, qlen;
    int kvh, krow, klen;
    int sees, n;             // keys that the tile works on, key tiles
    bool any;                // a row tile at all
};

__device__ __forceinline__ ShortItem short_item(const AttnArgs &A, int slots, int idx, int per) {
    ShortItem t;
    const int s = quotient(idx, A.heads), hx = idx - s * A.heads.d;
    // Later slots first: under a causal mask they see more keys.
    const Slot q = find_slot(A.q_off, A.k_off, A.n_seq, A.Tq, A.Tk, A.slot_rows, slots - 1 - s);
    t.any = q.first < q.len;
    t.kvh = hx / A.subs;
    t.qhead = t.kvh * (A.Hq / A.Hkv) + (hx % A.subs) * A.pack;
    t.qrow = q.base + q.first;
    t.tok0 = q.first;
    t.ntok = min(per, q.len - q.first);
    t.qlen = q.len;
    t.krow = q.other_base;
    t.klen = q.other_len;
    t.sees = A.causal ? min(t.klen, max(0, q.first + t.ntok + t.klen - q.len)) : t.klen;
    t.n = t.any ? (t.sees + ShortShape<32>::kKeys - 1) / ShortShape<32>::kKeys : 0;
    return t;
}

template <int DP>
__global__ void __launch_bounds__(128, ShortShape<DP>::kBlocks)
attn_forward_short_kernel(const AttnArgs A, const __grid_constant__ CUtensorMap mq,
                          const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                          const FwdOut f, int slots) {
    using S = ShortShape<DP>;
    using TL = Tile<DP>;
    constexpr int KEYS = S::kKeys;
    const uint32_t id_o = mma_idesc(128, (A.D + 15) & ~15, true);
    constexpr uint32_t kSbo = 8 * TL::kRowBytes, kQPanel = 128 * TL::kRowBytes, kPanel = KEYS * TL::kRowBytes;
    extern __shared__ unsigned char dyn[];
    __shared__ ShortShared sh;
    const int warp = warp_index();
    const bool boss = warp == 0;  // this warp also asks for copies and products
    const int per = 128 / A.pack;
    const int items = slots * A.heads.d;  // at most 2^31 - 1 by the launch

    if (boss) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.k_full[i], 1);
                mbar_init(&sh.v_full[i], 1);
            }
            mbar_init(&sh.s_full, 1);
            mbar_init(&sh.o_done, 1);
            mbar_init(&sh.drain, 1);
            sh.abort = 0;
            mbar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&sh.tmem, S::kTmem);
    }
    int idx = blockIdx.x;
    ShortItem it = short_item(A, slots, idx, per);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    const uint32_t smem_q = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t smem_k = smem_q + S::kQBytes, smem_v = smem_k + 2 * S::kTileBytes;
    volatile int *abort = &sh.abort;

    // Tiles of K and V are counted over all of the block's row tiles: the count says stage and phase.
    auto load_k = [&](const ShortItem &t, int g, int j, unsigned more) {
        mbar_arrive_expect_one(&sh.k_full[g & 1], S::kTileBytes + more);
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p)
            tma_load_3d_one(smem_k + (g & 1) * S::kTileBytes + p * kPanel, &mk, &sh.k_full[g & 1], p * TL::kCols, t.kvh,
                            t.krow + j * KEYS);
    };
    auto load_v = [&](const ShortItem &t, int g, int j) {
        mbar_arrive_expect_one(&sh.v_full[g & 1], S::kTileBytes);
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p)
            tma_load_3d_one(smem_v + (g & 1) * S::kTileBytes + p * kPanel, &mv, &sh.v_full[g & 1], p * TL::kCols, t.kvh,
                            t.krow + j * KEYS);
    };
    // The first tiles of a row tile whose count starts at g: Q with K's.
    auto load_first = [&](const ShortItem &t, int g) {
        load_k(t, g, 0, box_bytes<DP>(per * A.pack));
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p)
            tma_load_3d_one(smem_q + p * kQPanel, &mq, &sh.k_full[g & 1], p * TL::kCols, t.qhead, t.qrow);
        load_v(t, g, 0);
        if (t.n > 1) load_k(t, g + 1, 1, 0);
    };
    const uint64_t q_desc = smem_desc<TL::kRowBytes>(smem_q, 16, kSbo);
    const uint64_t k_desc = smem_desc<TL::kRowBytes>(smem_k, 16, kSbo);
    const uint64_t v_desc = smem_desc<TL::kRowBytes>(smem_v, kPanel, kSbo);
    auto scores = [&](int sees, int g, int j) {
        if (!wait_warp(&sh.k_full[g & 1], (g >> 1) & 1, abort)) return false;
        tc_fence_after();
        const uint32_t id = mma_idesc(128, tile_cols(sees, j * KEYS, KEYS), false);
        mma_channels<DP, kQPanel, kPanel>(tmem, q_desc, k_desc + (g & 1) * (S::kTileBytes / 16), id, A.D);
        tc_commit_one(&sh.s_full);
        return true;
    };

    const uint32_t ts = tmem + ((uint32_t)warp << 21), to = ts + KEYS;
    const int row = threadIdx.x, row_tok = row_token(A, row);
    int g = 0;                       // tiles of K and V before this row tile
    int k_asked = 0, v_asked = 0;    // warp 0: counts that copies were asked for
    unsigned done_phase = 0;
    bool ok = true, gave_up = false;
    if (boss && it.n > 0) {
        load_first(it, 0);
        k_asked = min(it.n, 2), v_asked = 1;
    }
#pragma unroll 1
    while (true) {
        if (boss && it.n > 0) ok = scores(it.sees, g, 0);
        // The next row tile, looked up while the tensor core starts on this one.
        idx = idx < items - (int)gridDim.x ? idx + (int)gridDim.x : items;
        ShortItem next;
        next.any = false;
        next.n = 0;
        if (idx < items) next = short_item(A, slots, idx, per);
        const bool live = it.any && row_tok < it.ntok;
        const bool warp_live = it.any && (row & ~31) < it.ntok * A.pack;
        const int limit = A.causal ? min(it.klen, max(0, it.tok0 + row_tok + 1 + it.klen - it.qlen)) : it.klen;
        const int all_see = A.causal ? min(it.klen, it.tok0 + 1 + it.klen - it.qlen) : it.klen;
        RowState rs(live);
#pragma unroll 1
        for (int i = 0; i < it.n; ++i) {
            const int t = g + i;
            ok = wait_warp(&sh.s_full, t & 1, abort) && ok;
            tc_fence_after();
            // S of this tile is done, and with it (in issue order) P V of the one before: K's buffer of this tile
            // and V's of the one before are free; after the last tile Q's and K's other buffer too.
            if (boss && ok) {
                if (i + 2 < it.n) load_k(it, t + 2, i + 2, 0), k_asked = t + 3;
                if (i + 1 < it.n) {
                    load_v(it, t + 1, i + 1), v_asked = t + 2;
                } else if (next.n > 0) {
                    load_first(next, t + 1);
                    k_asked = t + 1 + min(next.n, 2), v_asked = t + 2;
                }
            }
            const int k0 = i * KEYS;
            if (warp_live)
                softmax_tile64<DP>(rs, ts, to, tile_cols(it.sees, k0, KEYS), k0 + KEYS <= all_see, limit - k0, i == 0,
                                   A.scale_log2);
            // Rows of V that are not this sequence's (P is 0 there, but 0 x inf is not).
            if (k0 + KEYS > it.klen) {
                ok = wait_warp(&sh.v_full[t & 1], (t >> 1) & 1, abort) && ok;
                zero_rows<DP>(smem_v + (t & 1) * S::kTileBytes, KEYS, it.klen - k0, KEYS, 128);
                fence_async_smem();
            }
            tc_fence_before();
            gave_up = __syncthreads_or(!ok);
            if (gave_up) break;
            if (boss) {
                tc_fence_after();
                ok = wait_warp(&sh.v_full[t & 1], (t >> 1) & 1, abort);
                if (ok) {
                    const int steps = tile_cols(it.sees, k0, KEYS) / 16;
                    const uint64_t b = v_desc + (t & 1) * (S::kTileBytes / 16);
                    static_assert(KEYS == 64, "four steps");
                    if (steps == 4) {
                        mma_ts_one<4, TL::kRowBytes>(tmem + KEYS, tmem, b, id_o, i > 0);
                    } else {
#pragma unroll 1
                        for (int k = 0; k < steps; ++k)
                            mma_ts_one<1, 0>(tmem + KEYS, tmem + k * 8, b + k * TL::kRowBytes, id_o, i > 0 || k > 0);
                    }
                    if (i + 1 < it.n) ok = scores(it.sees, t + 1, i + 1);
                    else tc_commit_one(&sh.o_done);
                }
            }
        }
        if (gave_up) break;
        if (it.n > 0) {
            ok = wait_warp(&sh.o_done, done_phase, abort) && ok;
            done_phase ^= 1;
        } else if (boss && next.n > 0) {
            load_first(next, g);
            k_asked = g + min(next.n, 2), v_asked = g + 1;
        }
        tc_fence_after();
        // (O is written over only after the next row tile's first barrier.)
        if (ok && it.any)
            write_row<DP, false>(A, f, -1, rs, to, it.n > 0, live, (size_t)it.qrow + row_tok,
                                 it.qhead + row_head(A, row));
        tc_fence_before();
        g += it.n;
        if (idx >= items) break;
        it = next;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (boss) {
        if (sh.abort) {
            for (int i = max(0, k_asked - 2); i < k_asked; ++i)
                mbar_drain(&sh.k_full[i & 1], (i >> 1) & 1, kAttnWaitLimit);
            for (int i = max(0, v_asked - 2); i < v_asked; ++i)
                mbar_drain(&sh.v_full[i & 1], (i >> 1) & 1, kAttnWaitLimit);
            tc_commit_one(&sh.drain);
            mbar_drain(&sh.drain, 0, kAttnWaitLimit);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmem);
    }
}

// o = sum_s w_s part_s with w_s = exp(lse_s - lse), lse = log sum_s exp(lse_s), for a slot and head (x) whose keys
// were shared out; eight channels per thread.  A part that saw no keys has lse -inf, weight 0 and wrote zeros.
// Blocks look up their parts while the last of them are still in work, and read four parts at a time (weights
// relative to the largest lse so far).
__global__ void __launch_bounds__(128)
attn_join_kernel(const AttnArgs A, const FwdOut f, int slots, int least, int blocks) {
    __shared__ SharedOut so;
    count_tiles(A, so, slots);
    const unsigned size = share_size(A, so, slots, least, blocks);
    const int slot = quotient(blockIdx.x, A.heads), hx = blockIdx.x - slot * A.heads.d;
    const int parts = (so.tiles[slot] + size - 1) / size;
    int before = 0;
#pragma unroll 1
    for (int x = threadIdx.x & 31; x < slot; x += 32) before += (so.tiles[x] + size - 1) / size;
    before = __reduce_add_sync(0xffffffffu, before);
    // (One block at least waits, so that this launch does not end before the one whose parts it joins.)
    if (parts <= 1 && (blockIdx.x | blockIdx.y) > 0) return;
    wait_for_primary();
    if (parts <= 1) return;
    const Slot q = shared_slot(A, so, slot);
    const int per = 128 / A.pack, qhead = hx / A.subs * (A.Hq / A.Hkv) + (hx % A.subs) * A.pack;
    const int chunks = A.D / 8;
    const int rows = min(q.len - q.first, per) * A.pack;
    const size_t step = (size_t)A.heads.d * f.part_rows;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < rows * chunks; i += gridDim.y * blockDim.x) {
        const int row = i / chunks, c = (i - row * chunks) * 8;
        const size_t first = ((size_t)before * A.heads.d + hx) * f.part_rows + row;
        const float *pl = f.part_lse + first, *px = f.part + first * A.D + c;
        float top = -INFINITY, total = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
        for (int s = 0; s < parts; s += 4) {
            float l[4];
            float4 x[4][2];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool have = s + e < parts;
                const size_t at = (size_t)(s + e) * step;
                l[e] = have ? __ldcg(pl + at) : -INFINITY;
                x[e][0] = have ? __ldcg(reinterpret_cast<const float4 *>(px + at * A.D)) : make_float4(0, 0, 0, 0);
                x[e][1] = have ? __ldcg(reinterpret_cast<const float4 *>(px + at * A.D) + 1) : make_float4(0, 0, 0, 0);
            }
            const float was = top;
            top = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), was);
            const float ref = top == -INFINITY ? 0.0f : top, keep = expf(was - ref);
            total *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] *= keep;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = expf(l[e] - ref);
                total += w;
                o[0] = fmaf(w, x[e][0].x, o[0]);
                o[1] = fmaf(w, x[e][0].y, o[1]);
                o[2] = fmaf(w, x[e][0].z, o[2]);
                o[3] = fmaf(w, x[e][0].w, o[3]);
                o[4] = fmaf(w, x[e][1].x, o[4]);
                o[5] = fmaf(w, x[e][1].y, o[5]);
                o[6] = fmaf(w, x[e][1].z, o[6]);
                o[7] = fmaf(w, x[e][1].w, o[7]);
            }
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= inv;
        const size_t token = (size_t)q.base + q.first + row_token(A, row);
        const int head = qhead + row_head(A, row);
        store_result(f, (token * A.Hq + head) * A.D + c, o);
        if (f.lse && c == 0) f.lse[(size_t)head * A.Tq + token] = total == 0.0f ? -INFINITY : top + logf(total);
    }
}

// ---------------------------------------------------------------------------------------------
// Backward.
//
// Two kernels of one form, so that no sum needs an atomic and results do not depend on the order of
// blocks: one holds a tile of 128 keys (K, V) and walks the queries, accumulating dK and dV in
// TMEM; the other holds 128 query rows (Q, g) and walks the keys, accumulating dQ.  Both form S and
// dP again (three products where one kernel with atomics would share two of them).
//   X0, X1: the held tiles (K, V or Q, g); Y0, Y1: the walked ones, 64 or 32 rows a step (Q, g or K, V)
//   A = X0 Y0^T, B = X1 Y1^T  (128 x 64 or 32 each, TMEM)  ->  P = exp2(scale log2(e) A - log2(e) lse),
//   dS = P (B - delta)        (bf16, written over A and B)
//   acc0 += dS Y0             (dK or dQ, times scale at the end), acc1 += P Y1 (dV)
// With few held tiles (or, under a causal mask, one that walks far longer than the mean) a cluster of
// blocks shares a tile's steps; their accumulators are added through distributed shared memory, in
// rank order, each block writing its share of the columns.
// A warpgroup turns 32 columns of a pair (A, B) into P and dS.  64 rows a step, two warpgroups to a pair, is what
// TMEM leaves.  Up to 64 channels, one pair and two accumulators take half of it, and two blocks of an SM cover
// each other, their starts and ends too; up to 32, with 32 rows a step, a quarter, and four blocks do (104 x 300
// tokens of 8 heads of 32: 94 us for dK and dV, 62 for dQ, with 64 rows and two blocks 107 and 79).  With 128, two
// pairs alternate in one block: while one is in work, the tensor core forms the other and adds the one
// before.  (Two pairs in one block with 64 channels: 440 against 403 us for 4 x 2048 tokens of 12 heads, 392
// against 277 for 104 x 300 of 8 heads of 32, forward included.)
// What bounds it is the chain of a step, as forward: 8192 + 3001 + 130 causal tokens, 8 / 2 heads of 128, take
// 311 us for dK and dV (two blocks to a tile; four products a step) and 197 us for dQ (three), 1.0 and 1.2
// PFLOP/s of what they compute.
// P and dS are rounded to bf16 for the tensor core; every sum is float32.
// A row that sees exactly one key has P = 1 whatever its score, so its dS is set to what is left of
// it, the cotangent of its lse, rather than to the difference of two roundings of the same number.
// ---------------------------------------------------------------------------------------------
template <int DP> struct BwdShape {
    static constexpr int kWalk = DP == 32 ? 32 : 64;  // rows of Y a step
    static constexpr int kPairs = DP <= 64 ? 1 : 2;
    static constexpr int kXBytes = 128 * DP * 2;
    static constexpr int kYBytes = kWalk * DP * 2;
    static constexpr int kStages = 4;
    static constexpr int kHalves = kWalk / 32;  // warpgroups to a pair
    static constexpr int kCompute = kPairs * kHalves * 4;  // warps
    static constexpr int kThreads = kCompute * 32 + (DP == 32 ? 64 : 128);
    static constexpr int kBlocks = DP == 32 ? 4 : DP == 64 ? 2 : 1;
    // 65536 / 640 -> 96; 65536 / 768 -> 80.  (With 32 channels, 65536 / (4 x 192) -> 80 for all.)
    using Regs = std::conditional_t<kPairs == 2, Registers<4, 96, 104, 64>, Registers<2, 80, 96, 48>>;
    static constexpr int kTmem = 512 / kBlocks;
    static constexpr int kAcc = kPairs * 2 * kWalk;  // first accumulator column
    static_assert(kAcc + 2 * DP <= kTmem, "TMEM");
    static constexpr size_t kSmem = 1024 + 2 * kXBytes + (size_t)kStages * 2 * kYBytes;
};

struct BwdShared {
    uint64_t x_full, y_full[4], y_raw, y_empty[4], s_full[2], ds_ready[2], acc_done, drain;
    uint32_t tmem;
    int abort;
    // Per walked row, for the dK/dV kernel: -log2(e) lse, -delta and the lse's cotangent.
    alignas(16) float neg_lse2[4][64];
    alignas(16) float neg_delta[4][64];
    alignas(16) float one_ds[4][64];
    float row_dot[128];  // dQ: o.g of the held rows
};

// What both kernels know of the query rows.  The dQ kernel runs first and leaves delta = o.g - (the lse's
// cotangent) for the other; o is the output with what its rounding lost (with the rounded output alone dQ and
// dK were off by 1.5 to 1.6 times what plain bf16 calls are, with both by 1.4).  (With a kernel of its own for
// delta, and without the overlap of the two, 16 of 1 to 1601 tokens, 6 heads of 64, took 200 us both passes, now
// 189; 104 x 300, 8 of 32: 232 and 231.)
struct BwdRows {
    const bf16 *out, *low, *g;
    long long g_token, g_head;
    const float *lse, *g_lse;  // g_lse: or null
    float *delta;
};

// -log2(e) lse, for P = exp2(S' - lse').  A row whose scores are all -inf has lse -inf and, as forward, no weights:
// -inf too, where its negation would make them NaN.
__device__ __forceinline__ float neg_lse2(float lse) { return lse == -INFINITY ? -INFINITY : -lse * kLog2e; }

// What a block walks.  DKV: `steps_per_sub` tiles of `tok` tokens from token `first` on, for each of
// `subs` head groups.  DQ: tiles of 64 keys.
struct BwdRange {
    int steps, steps_per_sub;
    int start;      // this block's first step (its cluster's blocks share a tile's steps); steps ends them
    int first;      // DKV: first query token
    int qbase, qlen, kbase, klen;
    int tok;        // DKV: tokens a step
    int k0;         // DKV: first key of the held tile
    int q0, qtok;   // DQ: first token and tokens of the held tile
    int kvh, qhead; // key head; DQ: first query head of the tile (DKV: of the key head)
};

// Whole warp; returns how many steps were asked for.
template <int DP, bool DKV>
__device__ int bwd_load(const AttnArgs &A, const CUtensorMap *mx0, const CUtensorMap *mx1, const CUtensorMap *my0,
                        const CUtensorMap *my1, BwdShared &sh, uint32_t smem_x, uint32_t smem_y, const BwdRange &r,
                        const BwdRows &f) {
    using S = BwdShape<DP>;
    constexpr int kWalk = S::kWalk;
    using TL = Tile<DP>;
    const int lane = threadIdx.x & 31;
    volatile int *abort = &sh.abort;
    if (r.steps <= r.start) return 0;
    const int xrows = DKV ? 128 : (128 / A.pack) * A.pack;
    {
        mbar_arrive_expect_one(&sh.x_full, 2 * box_bytes<DP>(xrows));
        const int head = DKV ? r.kvh : r.qhead, at = DKV ? r.kbase + r.k0 : r.qbase + r.q0;
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p) {
            const uint32_t o = p * 128 * TL::kRowBytes;
            tma_load_3d_one(smem_x + o, mx0, &sh.x_full, p * TL::kCols, head, at);
            tma_load_3d_one(smem_x + S::kXBytes + o, mx1, &sh.x_full, p * TL::kCols, head, at);
        }
    }
    if (DKV) wait_for_primary();
    const int yrows = DKV ? r.tok * A.pack : kWalk;
    unsigned raw_phase = 0;
    int i = 0;
#pragma unroll 1
    for (; i < r.steps - r.start; ++i) {
        const int st = i % S::kStages;
        if (i >= S::kStages && !wait_warp(&sh.y_empty[st], ((i / S::kStages) - 1) & 1, abort)) break;
        const int step = r.start + i;
        const int sub = DKV ? step / r.steps_per_sub : 0;
        const int at = DKV ? r.first + (step - sub * r.steps_per_sub) * r.tok : step * kWalk;  // within the sequence
        const int head = DKV ? r.qhead + sub * A.pack : r.kvh;
        const int base = DKV ? r.qbase : r.kbase;
        // Rows of the box past the sequence's end belong to another sequence: cleared, since the
        // accumulating products multiply them by 0.
        const int good = DKV ? min(r.tok, r.qlen - at) * A.pack : min(kWalk, r.klen - at);
        uint64_t *bar = good < yrows ? &sh.y_raw : &sh.y_full[st];
        const uint32_t y0 = smem_y + st * 2 * S::kYBytes, y1 = y0 + S::kYBytes;
        mbar_expect_one(bar, 2 * box_bytes<DP>(yrows));
#pragma unroll
        for (int p = 0; p < TL::kPanels; ++p) {
            const uint32_t o = p * kWalk * TL::kRowBytes;
            tma_load_3d_one(y0 + o, my0, bar, p * TL::kCols, head, base + at);
            tma_load_3d_one(y1 + o, my1, bar, p * TL::kCols, head, base + at);
        }
        if (DKV) {
#pragma unroll
            for (int h = 0; h < kWalk / 32; ++h) {
                const int c = lane + h * 32;
                float nl = 0.0f, nd = 0.0f, od = 0.0f;
                if (c < good) {
                    const size_t x = (size_t)(head + row_head(A, c)) * A.Tq + base + at + row_token(A, c);
                    nl = neg_lse2(f.lse[x]);
                    nd = -__ldcg(f.delta + x);
                    if (f.g_lse) od = f.g_lse[x];
                }
                sh.neg_lse2[st][c] = nl;
                sh.neg_delta[st][c] = nd;
                sh.one_ds[st][c] = od;
            }
            __syncwarp();
        }
        mbar_arrive_one(bar);
        if (good < yrows) {
            if (!wait_warp(&sh.y_raw, raw_phase, abort)) {
                mbar_drain(&sh.y_raw, raw_phase, kAttnWaitLimit);
                break;
            }
            raw_phase ^= 1;
            zero_rows<DP>(y0, kWalk, good, yrows, 32);
            zero_rows<DP>(y1, kWalk, good, yrows, 32);
            fence_async_smem();
            __syncwarp();
            mbar_arrive_one(&sh.y_full[st]);
        }
    }
    return i;
}

// Whole warp.
template <int DP, bool DKV>
__device__ bool bwd_mma_loop(BwdShared &sh, uint32_t smem_x, uint32_t smem_y, int steps, uint32_t tmem, int dim) {
    using S = BwdShape<DP>;
    constexpr int kWalk = S::kWalk;
    using TL = Tile<DP>;
    constexpr uint32_t kIdS = mma_idesc(128, kWalk, false);
    const uint32_t id_acc = mma_idesc(128, (dim + 15) & ~15, true);
    constexpr uint32_t kSbo = 8 * TL::kRowBytes;
    constexpr uint32_t kXPanel = 128 * TL::kRowBytes, kYPanel = kWalk * TL::kRowBytes;
    volatile int *abort = &sh.abort;
    const uint64_t x_desc = smem_desc<TL::kRowBytes>(smem_x, 16, kSbo);
    const uint64_t y_desc = smem_desc<TL::kRowBytes>(smem_y, 16, kSbo);
    const uint64_t yt_desc = smem_desc<TL::kRowBytes>(smem_y, kYPanel, kSbo);
    auto scores = [&](int i) {
        const int st = i % S::kStages;
        if (!wait_warp(&sh.y_full[st], (i / S::kStages) & 1, abort)) return false;
        tc_fence_after();
        const uint64_t y = y_desc + st * (2 * S::kYBytes / 16);
#pragma unroll
        for (int which = 0; which < 2; ++which)
            mma_channels<DP, kXPanel, kYPanel>(tmem + (i % S::kPairs) * 2 * kWalk + which * kWalk,
                                               x_desc + which * (S::kXBytes / 16), y + which * (S::kYBytes / 16), kIdS,
                                               dim);
        tc_commit_one(&sh.s_full[i % S::kPairs]);
        return true;
    };
    if (!wait_warp(&sh.x_full, 0, abort)) return false;
    if (DKV) wait_for_primary();  // y_full comes after it
    if (!scores(0)) return false;
    if (S::kPairs == 2 && steps > 1 && !scores(1)) return false;
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
        const int st = i % S::kStages;
        const uint64_t y = yt_desc + st * (2 * S::kYBytes / 16);
        if (!wait_warp(&sh.ds_ready[i % S::kPairs], (i / S::kPairs) & 1, abort)) return false;
        tc_fence_after();
        const uint32_t p = tmem + (i % S::kPairs) * 2 * kWalk;
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
            const uint64_t yh = y + h * 2 * TL::kRowBytes;
            if (DKV)
                mma_ts_one<2, TL::kRowBytes>(tmem + S::kAcc + DP, p + h * 32, yh + S::kYBytes / 16, id_acc,
                                             i > 0 || h > 0);
            mma_ts_one<2, TL::kRowBytes>(tmem + S::kAcc, p + kWalk + h * 32, yh, id_acc, i > 0 || h > 0);
        }
        tc_commit_one(&sh.y_empty[st]);
        if (i + S::kPairs < steps && !scores(i + S::kPairs)) return false;
    }
    tc_commit_one(&sh.acc_done);
    return true;
}

// The kHalves warpgroups w: the steps i with i % kPairs == w, 32 columns each.
template <int DP, bool DKV>
__device__ void bwd_grads(const AttnArgs &A, BwdShared &sh, const BwdRange &r, uint32_t tmem, const BwdRows &f,
                          bool write_delta) {
    using S = BwdShape<DP>;
    constexpr int kWalk = S::kWalk;
    volatile int *abort = &sh.abort;
    const int group = threadIdx.x >> 7, w = group / S::kHalves, c0 = group % S::kHalves * 32, row = threadIdx.x & 127;
    const uint32_t ts = tmem + ((uint32_t)((threadIdx.x >> 5) & 3) << 21) + w * 2 * kWalk + c0;
    const float2 sc2 = make_float2(A.scale_log2, A.scale_log2);
    const int shift = r.klen - r.qlen;  // under a causal mask token t sees keys <= t + shift
    // DKV: this row's key.  DQ: this row's query.
    const int key = r.k0 + row;
    const int tok = r.q0 + row_token(A, row);
    int limit = 0;
    float row_nl = 0.0f, row_nd = 0.0f, row_od = 0.0f;
    if (!DKV) {
        // o.g of the held rows: DP / 8 lanes to a row, so that a warp's loads lie together (a thread to 32
        // channels of a row took 6 us a block with 128 channels).
        constexpr int kLanes = DP / 8, kRows = 32 / kLanes;
        static_assert(S::kCompute * 4 * kRows == 128, "four turns");
        const int lane = threadIdx.x & 31, c = lane % kLanes * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = ((threadIdx.x >> 5) * 4 + k) * kRows + lane / kLanes;
            float sum = 0.0f;
            if (row_token(A, at) < r.qtok && c < A.D) {
                const size_t token = (size_t)r.qbase + r.q0 + row_token(A, at);
                const int head = r.qhead + row_head(A, at);
                const size_t o = (token * A.Hq + head) * A.D + c;
                float a[8], b[8], l[8];
                load_vec<bf16, 8, true>(f.out + o, a);
                load_vec<bf16, 8, true>(f.low + o, l);
                load_vec<bf16, 8, true>(f.g + token * f.g_token + head * f.g_head + c, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(a[e], b[e], sum);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(l[e], b[e], sum);
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane % kLanes == 0) sh.row_dot[at] = sum;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(S::kCompute * 32) : "memory");
        if (row_token(A, row) < r.qtok) {
            limit = A.causal ? min(r.klen, max(0, tok + 1 + shift)) : r.klen;
            const size_t x = (size_t)(r.qhead + row_head(A, row)) * A.Tq + r.qbase + tok;
            row_nl = neg_lse2(f.lse[x]);
            if (f.g_lse) row_od = f.g_lse[x];
            row_nd = row_od - sh.row_dot[row];
            if (write_delta && group == 0) f.delta[x] = -row_nd;
        }
    }
    // DQ: keys that every row of the tile sees, and whether some row sees a single one.
    const int all_see = A.causal ? min(r.klen, r.q0 + 1 + shift) : r.klen;
    if (DKV) wait_for_primary();  // s_full comes after it
    // A warp without a live row leaves its rows of P and dS as they are: they reach no other row.
    const bool warp_live = DKV ? r.k0 + (row & ~31) < r.klen : (row & ~31) < r.qtok * A.pack;
#pragma unroll 1
    for (int i = w; i < r.steps - r.start; i += S::kPairs) {
        const int st = i % S::kStages;
        if (!wait_warp(&sh.s_full[w], (i / S::kPairs) & 1, abort)) return;
        if (!warp_live) {
            mbar_arrive_one(&sh.ds_ready[w]);
            continue;
        }
        tc_fence_after();
        // Of this thread's columns c0 ..: [lo, hi) of this row are seen; those in [one_lo, one_hi) belong to (DKV) or
        // the whole row is (DQ) a query with a single key.
        int lo = 0, hi = kWalk, one_lo = 0, one_hi = 0;
        bool mask;
        if (DKV) {
            const int at = r.first + ((r.start + i) % r.steps_per_sub) * r.tok;
            const int good = min(r.tok, r.qlen - at) * A.pack;
            mask = good < kWalk || r.k0 + 128 > r.klen || (A.causal && at + shift < r.k0 + 127);
            if (mask) {
                hi = key < r.klen ? good : 0;
                if (A.causal) {
                    lo = min(max(key - shift - at, 0), kWalk) * A.pack;
                    one_lo = min(max(-shift - at, -kWalk), kWalk) * A.pack;  // the token that sees key 0 only
                    one_hi = one_lo + A.pack;
                }
                if (r.klen == 1) {
                    one_lo = 0;
                    one_hi = kWalk;
                }
            }
        } else {
            mask = (r.start + i + 1) * kWalk > all_see;
            if (mask) {
                hi = limit - (r.start + i) * kWalk;
                one_hi = limit == 1 ? kWalk : 0;
            }
        }
        const uint32_t seen = bits(lo - c0, hi - c0), one = seen & bits(one_lo - c0, one_hi - c0);
        float s[32], d[32];
        tmem_ld32(ts, s);
        tmem_ld32(ts + kWalk, d);
        tmem_wait_ld();
        pin<32>(s);
        pin<32>(d);
        uint32_t ps[16], pd[16];
        // Straight code in either case: the exponentials' latencies overlap.
        auto weights = [&](auto masked) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            float4 nl, nd;
            if (DKV) {
                nl = *reinterpret_cast<const float4 *>(&sh.neg_lse2[st][c0 + c]);
                nd = *reinterpret_cast<const float4 *>(&sh.neg_delta[st][c0 + c]);
            } else {
                nl = make_float4(row_nl, row_nl, row_nl, row_nl);
                nd = make_float4(row_nd, row_nd, row_nd, row_nd);
            }
            const float2 a = fma2(make_float2(s[c], s[c + 1]), sc2, make_float2(nl.x, nl.y));
            const float2 b = fma2(make_float2(s[c + 2], s[c + 3]), sc2, make_float2(nl.z, nl.w));
            float p[4] = {exp2_fast(a.x), exp2_fast(a.y), exp2_fast(b.x), exp2_fast(b.y)};
            const float2 e = mul2(make_float2(p[0], p[1]), add2(make_float2(d[c], d[c + 1]), make_float2(nd.x, nd.y)));
            const float2 f =
                mul2(make_float2(p[2], p[3]), add2(make_float2(d[c + 2], d[c + 3]), make_float2(nd.z, nd.w)));
            float ds[4] = {e.x, e.y, f.x, f.y};
            if (masked) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t bit = 1u << (c + k);
                    p[k] = seen & bit ? p[k] : 0.0f;
                    ds[k] = seen & bit ? ds[k] : 0.0f;
                    if (masked == 2 && (one & bit)) ds[k] = DKV ? sh.one_ds[st][c0 + c + k] : row_od;
                }
            }
            ps[c / 2] = pack_bf16(p[0], p[1]);
            ps[c / 2 + 1] = pack_bf16(p[2], p[3]);
            pd[c / 2] = pack_bf16(ds[0], ds[1]);
            pd[c / 2 + 1] = pack_bf16(ds[2], ds[3]);
        }
        };
        if (!mask) weights(std::integral_constant<int, 0>{});
        else if (!__any_sync(0xffffffffu, one)) weights(std::integral_constant<int, 1>{});
        else weights(std::integral_constant<int, 2>{});
        // Over this half of A and B: the other half may not have been read yet.
        if (DKV) tmem_st16(ts, ps);
        tmem_st16(ts + kWalk, pd);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_one(&sh.ds_ready[w]);
    }
    if (r.steps > r.start) wait_warp(&sh.acc_done, 0, abort);
    tc_fence_after();
}

// Writes a row's part of the accumulators: the GROUPS warpgroups take 16 columns in turn.
template <int DP, bool DKV, int GROUPS>
__device__ __forceinline__ void store_acc(const AttnArgs &A, uint32_t acc, bool any, size_t row_at, bool live, bf16 *g0,
                                          bf16 *g1) {
    constexpr int kAll = DKV ? 2 * DP : DP;
#pragma unroll 1
    for (int c = (threadIdx.x >> 7) * 16; c < kAll; c += GROUPS * 16) {
        float o[16];
        if (any) {
            tmem_ld16(acc + c, o);
            tmem_wait_ld();
            pin<16>(o);
        }
        if (!live) continue;
        const bool second = DKV && c >= DP;
        const int col = second ? c - DP : c;
        const float f = second ? 1.0f : A.scale;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = any ? o[e] * f : 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 8)
            if (col + e < A.D) store_vec<bf16, 8>((second ? g1 : g0) + row_at + col + e, o + e);
    }
}

// Compute warps: this block's accumulator columns into its shared memory (column-major: a warp's rows are
// consecutive).
template <int DP, bool DKV, int GROUPS>
__device__ __forceinline__ void stage_acc(uint32_t acc, bool any, uint32_t smem) {
    constexpr int kAll = DKV ? 2 * DP : DP;
    const int w = threadIdx.x >> 7, row = threadIdx.x & 127;
#pragma unroll 1
    for (int c = w * 16; c < kAll; c += GROUPS * 16) {
        float o[16];
        if (any) {
            tmem_ld16(acc + c, o);
            tmem_wait_ld();
            pin<16>(o);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(smem + ((c + e) * 128 + row) * 4), "f"(any ? o[e] : 0.0f)
                         : "memory");
    }
}

// Whole block: the cluster's sums of this block's share of the columns to memory.
template <int DP, bool DKV, int GROUPS>
__device__ __forceinline__ void share_acc(const AttnArgs &A, uint32_t smem, int ranks, int rank, size_t row_at,
                                          bool live, bf16 *g0, bf16 *g1) {
    constexpr int kAll = DKV ? 2 * DP : DP;
    const int w = threadIdx.x >> 7, row = threadIdx.x & 127;
    cluster_sync();
    const int cols = kAll / ranks;
    if (w < GROUPS) {
#pragma unroll 1
        for (int c = rank * cols + w * 8; c < (rank + 1) * cols; c += GROUPS * 8) {
            float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
            for (int k = 0; k < ranks; ++k) {
                const uint32_t from = cluster_addr(smem + (c * 128 + row) * 4, k);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += cluster_ld(from + e * 512);
            }
            const bool second = DKV && c >= DP;
            const int col = second ? c - DP : c;
            if (live && col < A.D) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= second ? 1.0f : A.scale;
                store_vec<bf16, 8>((second ? g1 : g0) + row_at + col, o);
            }
        }
    }
    cluster_sync();  // no block leaves while another reads its shared memory
}

template <int DP, bool DKV>
__global__ void __launch_bounds__(BwdShape<DP>::kThreads, BwdShape<DP>::kBlocks)
attn_backward_kernel(const AttnArgs A, const __grid_constant__ CUtensorMap mx0, const __grid_constant__ CUtensorMap mx1,
                     const __grid_constant__ CUtensorMap my0, const __grid_constant__ CUtensorMap my1,
                     const BwdRows f, bf16 *__restrict__ g0, bf16 *__restrict__ g1, int slots, int ranks) {
    using S = BwdShape<DP>;
    constexpr int kWalk = S::kWalk;
    extern __shared__ unsigned char dyn[];
    __shared__ __align__(16) BwdShared sh;
    const int warp = warp_index();
    const int log_ranks = __popc(ranks - 1);  // 1, 2 or 4
    const int rank = blockIdx.x & (ranks - 1), tile = blockIdx.x >> log_ranks;
    const int s = quotient(tile, A.heads), hx = tile - s * A.heads.d;
    // The tiles with most work under a causal mask first: the first keys, the last queries.
    const int slot = DKV ? s : slots - 1 - s;
    const int per = DKV ? 128 : 128 / A.pack;
    const Slot x = DKV ? find_slot(A.k_off, A.q_off, A.n_seq, A.Tk, A.Tq, A.slot_rows, slot)
                       : find_slot(A.q_off, A.k_off, A.n_seq, A.Tq, A.Tk, A.slot_rows, slot);
    // The dK/dV launch overlaps the dQ one's end: its warps wait for delta, and its first block at least, so that it
    // does not end before the other.
    if (DKV && blockIdx.x == 0) wait_for_primary();
    if (x.first >= x.len) return;
    const int G = A.Hq / A.Hkv;
    BwdRange r;
    r.kvh = DKV ? hx : hx / A.subs;
    r.qhead = r.kvh * G + (DKV ? 0 : (hx % A.subs) * A.pack);
    r.tok = kWalk / A.pack;
    r.first = r.k0 = r.q0 = r.qtok = 0;
    r.steps_per_sub = 1;
    if (DKV) {
        r.kbase = x.base, r.klen = x.len, r.k0 = x.first;
        r.qbase = x.other_base, r.qlen = x.other_len;
        r.first = A.causal ? min(r.qlen, max(0, r.k0 + r.qlen - r.klen)) : 0;
        r.steps_per_sub = (r.qlen - r.first + r.tok - 1) / r.tok;
        r.steps = r.steps_per_sub * A.subs;
    } else {
        r.qbase = x.base, r.qlen = x.len, r.q0 = x.first;
        r.kbase = x.other_base, r.klen = x.other_len;
        r.qtok = min(per, r.qlen - r.q0);
        const int sees = A.causal ? min(r.klen, max(0, r.q0 + r.qtok + r.klen - r.qlen)) : r.klen;
        r.steps = (sees + kWalk - 1) / kWalk;
    }
    const int each = (r.steps + ranks - 1) / ranks;
    r.start = min(r.steps, each * rank);
    r.steps = min(r.steps, r.start + each);
    const int steps = r.steps - r.start;
    const uint32_t smem_x = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t smem_y = smem_x + 2 * S::kXBytes;

    if (warp == S::kCompute) {
        if ((threadIdx.x & 31) == 0) {
            mbar_init(&sh.x_full, 1);
            for (int i = 0; i < S::kStages; ++i) {
                mbar_init(&sh.y_full[i], 1);
                mbar_init(&sh.y_empty[i], 1);
            }
            mbar_init(&sh.y_raw, 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&sh.s_full[b], 1);
                mbar_init(&sh.ds_ready[b], S::kHalves * 4);
            }
            mbar_init(&sh.acc_done, 1);
            mbar_init(&sh.drain, 1);
            sh.abort = 0;
            mbar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&sh.tmem, S::kTmem);
    }
    // Rows of a step that no box ever fills (heads that do not divide a step) must hold numbers.
    if (DKV && r.tok * A.pack < kWalk) {
        for (int i = threadIdx.x; i < S::kStages * 2 * S::kYBytes / 16; i += S::kThreads)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_y + i * 16), "r"(0) : "memory");
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    // Only now that this block has its TMEM: a dK/dV block holds its own until all of this launch has ended, so one
    // let in before could keep a block of this launch waiting for the columns that it holds.
    if (!DKV) launch_dependents();

    int issued = 0;
    const int row = threadIdx.x & 127;
    const uint32_t acc = tmem + ((uint32_t)(warp & 3) << 21) + S::kAcc;
    const bool live = DKV ? r.k0 + row < r.klen : row_token(A, row) < r.qtok;
    const size_t row_at = DKV ? ((size_t)(r.kbase + r.k0 + row) * A.Hkv + r.kvh) * A.D
                              : ((size_t)(r.qbase + r.q0 + row_token(A, row)) * A.Hq + r.qhead + row_head(A, row)) *
                                    A.D;
    if (warp >= S::kCompute) {
        if constexpr (DP > 32) regs_less<S::Regs::kLess>();
        if (warp == S::kCompute && steps > 0) bwd_mma_loop<DP, DKV>(sh, smem_x, smem_y, steps, tmem, A.D);
        if (warp == S::kCompute + 1)
            issued = bwd_load<DP, DKV>(A, &mx0, &mx1, &my0, &my1, sh, smem_x, smem_y, r, f);
    } else {
        if constexpr (DP > 32) regs_more<S::Regs::kMore>();
        bwd_grads<DP, DKV>(A, sh, r, tmem, f, rank == 0);
        __syncwarp();
        if (ranks == 1) store_acc<DP, DKV, S::kCompute / 4>(A, acc, steps > 0, row_at, live, g0, g1);
    }
    if (ranks > 1) {
        // Every product of this block is done, so its shared memory is free.
        __syncthreads();
        if (warp < S::kCompute) stage_acc<DP, DKV, S::kCompute / 4>(acc, steps > 0, smem_x);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (sh.abort && warp == S::kCompute + 1 && (threadIdx.x & 31) == 0 && steps > 0) {
        mbar_drain(&sh.x_full, 0, kAttnWaitLimit);
        for (int i = max(0, issued - S::kStages); i < issued; ++i)
            mbar_drain(&sh.y_full[i % S::kStages], (i / S::kStages) & 1, kAttnWaitLimit);
    }
    if (warp == S::kCompute) {
        if (sh.abort) {
            tc_commit_one(&sh.drain);
            mbar_drain(&sh.drain, 0, kAttnWaitLimit);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmem);
    }
    // The block gives its TMEM back before it waits for the cluster's others: one of them may still be waiting for
    // TMEM on its own SM, held there by a block that waits for one more.
    if (ranks > 1) {
        __syncwarp();
        share_acc<DP, DKV, S::kCompute / 4>(A, smem_x, ranks, rank, row_at, live, g0, g1);
    }
}

// ---------------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------------

// The largest divisor of the group that is at most `most`.
int pack_of(long long group, int most) {
    for (int p = (int)(group < most ? group : most); p > 1; --p)
        if (group % p == 0) return p;
    return 1;
}

int padded_dim(long long D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct Strided {
    const void *p;
    int64_t token, head;  // strides in elements
};

// Boxes of `heads` x `tokens` rows, one column panel wide.
bool make_map(CUtensorMap *map, const Strided &t, long long T, long long H, long long D, int heads, int tokens,
              const void *spare) {
    const int cols = D <= 32 ? 32 : 64;
    uint64_t dims[3] = {(uint64_t)D, (uint64_t)H, (uint64_t)(T > 0 ? T : 1)};
    uint64_t strides[2] = {(uint64_t)t.head * 2, (uint64_t)t.token * 2};
    const void *base = t.p;
    if (T == 0) {  // never loaded from; any valid description does
        strides[0] = strides[1] = 16;
        dims[0] = 8;
        dims[1] = 1;
        base = spare;
    }
    const uint32_t box[3] = {(uint32_t)cols, (uint32_t)heads, (uint32_t)tokens};
    return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box,
                             cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename K> int allow_smem(K kernel, size_t bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess
               ? RFDETR_OK
               : RFDETR_ERR_CUDA;
}

constexpr long long kMaxRows = 1ll << 30;  // rows and offsets are int32 in the kernels

int check_sizes(int64_t n_seq, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hkv, int64_t D) {
    if (n_seq < 0 || n_seq > kMaxRows || Tq < 0 || Tq > kMaxRows || Tk < 0 || Tk > kMaxRows) return RFDETR_ERR_SHAPE;
    if (Hkv < 1 || Hq < Hkv || Hq > 65536 || Hq % Hkv) return RFDETR_ERR_SHAPE;
    if (D < 8 || D > 128 || D % 8) return RFDETR_ERR_SHAPE;
    return RFDETR_OK;
}

int check_tensor(const Strided &t, int64_t T, int64_t H) {
    if (T == 0) return RFDETR_OK;
    if (!t.p || !aligned(t.p, 16)) return RFDETR_ERR_ALIGN;
    // Strides of a size-1 axis do not matter to the caller, but the tensor map wants them valid.
    if (t.token <= 0 || t.head <= 0 || t.token % 8 || t.head % 8) return RFDETR_ERR_ALIGN;
    if (t.token >= (1ll << 38) || t.head >= (1ll << 38)) return RFDETR_ERR_SHAPE;
    (void)H;
    return RFDETR_OK;
}

// Which forward kernel, and whether the row tiles' keys are shared out over blocks.
struct ForwardPlan {
    bool is_short;
    bool alternate;  // one row tile a block, its key tiles taken by the block's halves in turn
    int blocks;      // that the keys are shared out over (alternate only); 0: one block to a slot and head
    int slot_rows;
    long long slots;
};

ForwardPlan plan_forward(const AttnArgs &A) {
    const int per = 128 / A.pack, sms = num_sms();
    const long long heads = (long long)A.Hkv * A.subs;
    const long long n_seq = A.n_seq > 0 ? A.n_seq : 1;
    const long long rows = A.Tq / n_seq, keys = A.Tk / n_seq, tiles = (keys + 127) / 128;  // of the mean sequence
    // Row tiles, and pairs of them, if every sequence were the mean one.
    const long long row_tiles = heads * n_seq * ((rows + per - 1) / per);
    const long long pairs = heads * n_seq * ((rows + 2 * per - 1) / (2 * per));
    const bool single = rows <= per;
    ForwardPlan p{};
    // (us, the alternating halves against pairs of row tiles; tokens x heads of channels.)  One to an SM at most:
    // 300 tokens, 8 of 32: 9.3, 11.0; 4 x 577, 6 of 64: 12.5, 16.6; 1024 causal, 16 / 4 of 128: 16.6, 22.7; 4 x
    // 300 over 2000 keys, 8 of 64: 20.7, 32.9; but 8 x 577, 6 of 64, 240 row tiles: 22.7, 18.6.  With more, for
    // long keys:
    // * under a causal mask up to one and a half an SM (the longest begin first): 2 x 1601, 8 of 64: 19.7, 26.4; 1601,
    //   16 / 4 of 128: 21.4, 28.0; 4 x 1024, 6 of 64: 18.9, 19.7; and with ten key tiles up to two: 2048, 16 / 4 of
    //   128: 27.4, 34.1; 2 x 3000, 6 of 64: 32, 46.5; 2 x 1300, 12 of 64: 21.7, 23.6; but 4 x 1024, 8 of 64, 256 row
    //   tiles of eight: 21.4, 19.6; 6 x 900, 6 of 64: 22.6, 19.6;
    // * up to one and a half where the keys are other tokens and there are several sequences.  Whether the keys' counts
    //   differ the host does not know; where they do, halves take 0.8 of the time in the mean of 135 sizes (0.47 to
    //   1.2; 8 x 300 over 0 to 4000, 8 of 80: 32.6, 57.1; over 700 to 3200: 28.9, 48.1), where they are equal 1.04
    //   with up to 64 channels and 1.17 with more (45 sizes; 8 x 300 over 2000 each, 8 of 64: 35.7, 34.2; of 80:
    //   38.9, 33.8).  A single sequence has one count, and pairs: 3000 over 2000, 8 of 80: 39.0, 33.7;
    // * where a pair's second would be empty: 24 x 100 over 1000, 8 of 32: 23.1, 28.2; 128 x 1 over 2000, 16 / 4 of
    //   128: 108.7, 117.6; 32 x 1 over 700, 8 of 64: 25.0, 28.2.
    const bool unequal = A.Tq != A.Tk && n_seq > 1;  // as far as can be told
    p.alternate = tiles >= 2 && (row_tiles <= sms ||
                                 (tiles >= 8 && (single || ((A.causal || unequal) && 2 * row_tiles <= 3 * sms))) ||
                                 (tiles >= 10 && A.causal && row_tiles <= 2 * sms));
    // Shared out over the SMs, a block to each: one token over 30,000 keys, 32 / 8 of 128: 38.4, whole 220; 4 x 64
    // over 8000, 16 / 4: 39.3, 68.1; 4 x 1 over 2500, 8 of 64: 18.6, 22.7; but 16 x 1 over 4000, 16 / 4: 36.7,
    // 41.7; 1601, 6 of 64, 13 key tiles: 29.3, 18.6.
    bool share = p.alternate && tiles >= 16 && 2 * row_tiles <= sms;
    long long times = 0;
    // The short kernel against pairs of row tiles: 104 x 300, 8 of 32: 57, 103; 32 x 145, 6 of 64: 12.0, 16.2; 16
    // x 64, 4 of 64: 6.3, 8.4; 16 x 300 over 1000, 8 of 32: 35.0, 39.6; but 8 x 300, 8 of 32, 128 pairs: 14.5,
    // 12.5; 16 of 1 to 1601, 6 of 64: 54.7, 53.2.  (Single tokens, against halves: 32 x 1 over 700, 8 of 64: 22.7,
    // 25.0; over 1500: 41.2, 37.1.)
    p.is_short = !p.alternate && rows <= 4 * per &&
                 (keys <= 128 || (pairs > sms && keys <= 512) || (single && tiles < 8));
    const KnobValue forced = knob(kKnobAttnFwd);
    if (forced.count > 0 && forced.v[0] > 0) {
        p.is_short = forced.v[0] == 2;
        p.alternate = forced.v[0] == 3;
        times = !p.alternate || forced.v[1] < 2 ? 0 : forced.v[1] > 64 ? 64 : forced.v[1];
        share = times > 0;
    }
    p.slot_rows = p.is_short || p.alternate ? per : per * 2;
    p.slots = slots_for(A.Tq, p.slot_rows, A.n_seq);
    if (share && p.slots <= kSharedSlots) {
        const long long most = p.slots * heads;
        p.blocks = (int)(times > 0 ? most * times : most > sms ? most : sms);
    }
    return p;
}

int part_rows(const AttnArgs &A) {
    const int per = 128 / A.pack;
    return (A.Tq < per ? A.Tq : per) * A.pack;
}
size_t split_bytes(const AttnArgs &A, const ForwardPlan &p) {
    return (size_t)p.blocks * part_rows(A) * (A.D + 1) * sizeof(float);
}

template <int DP>
int launch_forward(AttnArgs A, const ForwardPlan &plan, const Strided &q, const Strided &k, const Strided &v,
                   const FwdOut &f, cudaStream_t stream) {
    const int per = 128 / A.pack, keys = plan.is_short ? ShortShape<DP>::kKeys : LongShape<DP, false>::kKeys;
    CUtensorMap mq, mk, mv;
    if (!make_map(&mq, q, A.Tq, A.Hq, A.D, A.pack, per, q.p) || !make_map(&mk, k, A.Tk, A.Hkv, A.D, 1, keys, q.p) ||
        !make_map(&mv, v, A.Tk, A.Hkv, A.D, 1, keys, q.p))
        return RFDETR_ERR_CUDA;
    const long long blocks = plan.slots * A.Hkv * A.subs;
    if (blocks > 0x7fffffffll) return RFDETR_ERR_SHAPE;
    const int slots = (int)plan.slots;
    A.slot_rows = divisor(plan.slot_rows);
    A.heads = divisor(A.Hkv * A.subs);
    if (plan.is_short) {
        using S = ShortShape<DP>;
        const long long stay = (long long)S::kBlocks * num_sms();
        if (int st = allow_smem(attn_forward_short_kernel<DP>, S::kSmem)) return st;
        attn_forward_short_kernel<DP>
            <<<(unsigned)(blocks < stay ? blocks : stay), 128, S::kSmem, stream>>>(A, mq, mk, mv, f, slots);
        return launch_status();
    }
    using S = LongShape<DP, false>;  // (its block and shared memory are those of the alternating kernel too)
    auto launch = [&](auto kernel) {
        if (int st = allow_smem(kernel, S::kSmem)) return st;
        const unsigned grid = (unsigned)(plan.blocks ? plan.blocks : blocks);
        kernel<<<grid, S::kThreads, S::kSmem, stream>>>(A, mq, mk, mv, f, slots);
        return launch_status();
    };
    if (plan.blocks == 0)
        return plan.alternate ? launch(attn_forward_long_kernel<DP, true, false>)
                              : launch(attn_forward_long_kernel<DP, false, false>);
    if (int st = launch(attn_forward_long_kernel<DP, true, true>)) return st;
    const int most = A.Tq < plan.slot_rows ? A.Tq : plan.slot_rows;  // tokens of a slot
    cudaLaunchConfig_t config{};
    const int items = most * A.pack * (A.D / 8), threads = items <= 512 ? 32 : 128;
    const int chunks = (items + threads - 1) / threads;
    config.gridDim = dim3((unsigned)blocks, (unsigned)(chunks < 16 ? chunks : 16));
    config.blockDim = dim3((unsigned)threads);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, attn_join_kernel, A, f, slots, S::kLeast, plan.blocks) != cudaSuccess) {
        (void)cudaGetLastError();
        return RFDETR_ERR_CUDA;
    }
    return RFDETR_OK;
}

// Blocks that share a held tile's steps, in the kernel that holds keys and in the one that holds
// queries.
struct BackwardPlan {
    int kv_ranks, q_ranks;
};

template <int DP> BackwardPlan plan_backward(const AttnArgs &A) {
    using S = BwdShape<DP>;
    const long long n_seq = A.n_seq > 0 ? A.n_seq : 1;
    const long long rows = (A.Tq + n_seq - 1) / n_seq, keys = (A.Tk + n_seq - 1) / n_seq;  // of the mean sequence
    const int per = 128 / A.pack;
    // While each has an SM of its own, down to four steps a block; with many steps, up to four an SM.  (us, tokens x
    // heads of channels, alone and shared by so many for keys, queries: 300, 8 of 32: 26.8, 22.7 by 2, 2; 577, 6 of
    // 64: 34.9, 28.8 by 2, 2; 1000 causal, 8 of 128: 41.2, 35.0 by 2, 2 and 55.5 by 4, 4; 2048, 8 of 32: 112.8, 70.2 by
    // 4, 4; but 300, 8 of 128, four steps: 24.8, 26.7 by 2, 2; 4 x 577, 120 tiles: 37.0, 43.0 by 1, 2.)
    auto ranks = [&](long long blocks, long long steps) {
        const long long sms = num_sms();
        int r = 1;
        while (r < 4 && ((blocks * 2 * r <= sms && steps >= 8 * r) || (blocks * r < 2 * sms && steps >= 16 * r))) r *= 2;
        return r;
    };
    BackwardPlan p;
    p.kv_ranks = ranks(n_seq * A.Hkv * ((keys + 127) / 128), rows * A.pack * A.subs / S::kWalk);
    p.q_ranks = ranks(n_seq * A.Hkv * A.subs * ((rows + per - 1) / per), keys / S::kWalk);
    const KnobValue forced = knob(kKnobAttnBwd);
    auto valid = [](int r) { return r == 1 || r == 2 || r == 4; };
    if (forced.count > 0 && valid(forced.v[0])) p.kv_ranks = forced.v[0];
    if (forced.count > 1 && valid(forced.v[1])) p.q_ranks = forced.v[1];
    return p;
}

template <int DP, bool DKV, typename... Args>
int launch_backward_kernel(long long tiles, int ranks, bool overlap, cudaStream_t stream, Args... args) {
    using S = BwdShape<DP>;
    if (tiles * ranks > 0x7fffffffll) return RFDETR_ERR_SHAPE;
    if (int st = allow_smem(attn_backward_kernel<DP, DKV>, S::kSmem)) return st;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(tiles * ranks));
    config.blockDim = dim3(S::kThreads);
    config.dynamicSmemBytes = S::kSmem;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    config.attrs = attr;
    if (ranks > 1) {
        attr[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[config.numAttrs++].val.clusterDim = {(unsigned)ranks, 1, 1};
    }
    if (overlap) {
        attr[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cudaLaunchKernelEx(&config, attn_backward_kernel<DP, DKV>, args..., ranks) != cudaSuccess) {
        (void)cudaGetLastError();
        return RFDETR_ERR_CUDA;
    }
    return RFDETR_OK;
}

template <int DP>
int launch_backward(AttnArgs A, const Strided &q, const Strided &k, const Strided &v, const Strided &g,
                    const BwdRows &f, bf16 *dq, bf16 *dk, bf16 *dv, cudaStream_t stream) {
    constexpr int kWalk = BwdShape<DP>::kWalk;
    const BackwardPlan plan = plan_backward<DP>(A);
    CUtensorMap kx, vx, qy, gy, qx, gx, ky, vy;
    const int ytok = kWalk / A.pack, xtok = 128 / A.pack;
    if (!make_map(&kx, k, A.Tk, A.Hkv, A.D, 1, 128, q.p) || !make_map(&vx, v, A.Tk, A.Hkv, A.D, 1, 128, q.p) ||
        !make_map(&ky, k, A.Tk, A.Hkv, A.D, 1, kWalk, q.p) || !make_map(&vy, v, A.Tk, A.Hkv, A.D, 1, kWalk, q.p) ||
        !make_map(&qy, q, A.Tq, A.Hq, A.D, A.pack, ytok, k.p) ||
        !make_map(&gy, g, A.Tq, A.Hq, A.D, A.pack, ytok, k.p) ||
        !make_map(&qx, q, A.Tq, A.Hq, A.D, A.pack, xtok, k.p) ||
        !make_map(&gx, g, A.Tq, A.Hq, A.D, A.pack, xtok, k.p))
        return RFDETR_ERR_CUDA;
    if (A.Tq > 0) {
        const long long slots = slots_for(A.Tq, xtok, A.n_seq), blocks = slots * A.Hkv * A.subs;
        A.slot_rows = divisor(xtok);
        A.heads = divisor(A.Hkv * A.subs);
        if (int st = launch_backward_kernel<DP, false>(blocks, plan.q_ranks, false, stream, A, qx, gx, ky, vy, f, dq,
                                                       nullptr, (int)slots))
            return st;
    }
    if (A.Tk > 0) {
        const long long slots = slots_for(A.Tk, 128, A.n_seq), blocks = slots * A.Hkv;
        A.slot_rows = divisor(128);
        A.heads = divisor(A.Hkv);
        if (int st = launch_backward_kernel<DP, true>(blocks, plan.kv_ranks, A.Tq > 0, stream, A, kx, vx, qy, gy, f, dk,
                                                      dv, (int)slots))
            return st;
    }
    return RFDETR_OK;
}

AttnArgs make_args(const int32_t *q_off, const int32_t *k_off, int64_t n_seq, int64_t Tq, int64_t Tk, int64_t Hq,
                   int64_t Hkv, int64_t D, int causal, float scale, int most_packed) {
    AttnArgs A;
    A.q_off = q_off;
    A.k_off = k_off ? k_off : q_off;
    A.n_seq = (int)n_seq;
    A.Tq = (int)Tq;
    A.Tk = (int)Tk;
    A.Hq = (int)Hq;
    A.Hkv = (int)Hkv;
    A.D = (int)D;
    A.pack = pack_of(Hq / Hkv, most_packed);
    A.pack_inv = (65536 + A.pack - 1) / A.pack;
    A.subs = (int)(Hq / Hkv) / A.pack;
    A.causal = causal != 0;
    A.scale = scale;
    A.scale_log2 = scale * kLog2e;
    return A;
}

}  // namespace

// Reads and clears this file's device fault word; bits are those of mbar_wait / mbar_drain.
int take_attention_fault(cudaStream_t stream, unsigned *word) {
    void *p = nullptr;
    if (cudaGetSymbolAddress(&p, g_device_fault) != cudaSuccess) return RFDETR_ERR_CUDA;
    if (cudaMemcpyAsync(word, p, sizeof(unsigned), cudaMemcpyDeviceToHost, stream) != cudaSuccess)
        return RFDETR_ERR_CUDA;
    if (cudaMemsetAsync(p, 0, sizeof(unsigned), stream) != cudaSuccess) return RFDETR_ERR_CUDA;
    return cudaStreamSynchronize(stream) == cudaSuccess ? RFDETR_OK : RFDETR_ERR_CUDA;
}

}  // namespace rfdetr

extern "C" size_t rfdetr_packed_attention_workspace_bytes(int64_t n_sequences, int64_t tokens, int64_t key_tokens,
                                                          int64_t n_heads, int64_t n_kv_heads, int64_t head_dim) {
    using namespace rfdetr;
    if (check_sizes(n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim) != RFDETR_OK) return 0;
    const AttnArgs A = make_args(nullptr, nullptr, n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim, 0,
                                 1.0f, 128);
    return split_bytes(A, plan_forward(A));
}

extern "C" int rfdetr_packed_attention(void *stream, const void *query, int64_t query_token_stride,
                                       int64_t query_head_stride, const void *key, int64_t key_token_stride,
                                       int64_t key_head_stride, const void *value, int64_t value_token_stride,
                                       int64_t value_head_stride, const int32_t *offsets, const int32_t *key_offsets,
                                       void *output, void *output_low, float *lse, void *workspace,
                                       size_t workspace_bytes,
                                       int64_t n_sequences, int64_t tokens, int64_t key_tokens, int64_t n_heads,
                                       int64_t n_kv_heads, int64_t head_dim, int causal, float scale) {
    using namespace rfdetr;
    if (int st = check_sizes(n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim)) return st;
    if (!(scale > 0.0f) || scale > FLT_MAX) return RFDETR_ERR_SHAPE;
    if (tokens == 0) return RFDETR_OK;
    const Strided q{query, query_token_stride, query_head_stride}, k{key, key_token_stride, key_head_stride},
        v{value, value_token_stride, value_head_stride};
    if (int st = check_tensor(q, tokens, n_heads)) return st;
    if (int st = check_tensor(k, key_tokens, n_kv_heads)) return st;
    if (int st = check_tensor(v, key_tokens, n_kv_heads)) return st;
    if (!output || !aligned(output, 16) || !aligned(output_low, 16) || !aligned(lse, 4) || !offsets ||
        !aligned(offsets, 4) || !aligned(key_offsets, 4))
        return RFDETR_ERR_ALIGN;
    const AttnArgs A = make_args(offsets, key_offsets, n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim,
                                 causal, scale, 128);
    const ForwardPlan p = plan_forward(A);
    const size_t need = split_bytes(A, p);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return RFDETR_ERR_WORKSPACE;
    FwdOut f{static_cast<bf16 *>(output), static_cast<bf16 *>(output_low), lse};
    if (need) {
        f.part = static_cast<float *>(workspace);
        f.part_rows = part_rows(A);
        f.part_lse = f.part + (size_t)p.blocks * f.part_rows * A.D;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (padded_dim(head_dim)) {
        case 32: return launch_forward<32>(A, p, q, k, v, f, s);
        case 64: return launch_forward<64>(A, p, q, k, v, f, s);
        default: return launch_forward<128>(A, p, q, k, v, f, s);
    }
}

extern "C" size_t rfdetr_packed_attention_backward_workspace_bytes(int64_t tokens, int64_t n_heads) {
    if (tokens < 0 || tokens > rfdetr::kMaxRows || n_heads < 0 || n_heads > 65536) return 0;
    return (size_t)tokens * n_heads * sizeof(float);
}

extern "C" int rfdetr_packed_attention_backward(
    void *stream, const void *query, int64_t query_token_stride, int64_t query_head_stride, const void *key,
    int64_t key_token_stride, int64_t key_head_stride, const void *value, int64_t value_token_stride,
    int64_t value_head_stride, const int32_t *offsets, const int32_t *key_offsets, const void *output,
    const void *output_low, const float *lse, const void *grad_output, int64_t grad_token_stride,
    int64_t grad_head_stride,
    const float *grad_lse, void *grad_query, void *grad_key, void *grad_value, void *workspace, size_t workspace_bytes,
    int64_t n_sequences, int64_t tokens, int64_t key_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
    int causal, float scale) {
    using namespace rfdetr;
    if (int st = check_sizes(n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim)) return st;
    if (!(scale > 0.0f) || scale > FLT_MAX) return RFDETR_ERR_SHAPE;
    if (tokens == 0 && key_tokens == 0) return RFDETR_OK;
    const Strided q{query, query_token_stride, query_head_stride}, k{key, key_token_stride, key_head_stride},
        v{value, value_token_stride, value_head_stride}, g{grad_output, grad_token_stride, grad_head_stride};
    if (int st = check_tensor(q, tokens, n_heads)) return st;
    if (int st = check_tensor(g, tokens, n_heads)) return st;
    if (int st = check_tensor(k, key_tokens, n_kv_heads)) return st;
    if (int st = check_tensor(v, key_tokens, n_kv_heads)) return st;
    if (!offsets || !aligned(offsets, 4) || !aligned(key_offsets, 4)) return RFDETR_ERR_ALIGN;
    if (tokens > 0 && (!output || !aligned(output, 16) || !output_low || !aligned(output_low, 16) || !grad_query ||
                       !aligned(grad_query, 16) || !lse || !aligned(lse, 4) || !aligned(grad_lse, 4)))
        return RFDETR_ERR_ALIGN;
    if (key_tokens > 0 && (!grad_key || !grad_value || !aligned(grad_key, 16) || !aligned(grad_value, 16)))
        return RFDETR_ERR_ALIGN;
    const size_t need = rfdetr_packed_attention_backward_workspace_bytes(tokens, n_heads);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 4))) return RFDETR_ERR_WORKSPACE;
    const AttnArgs A = make_args(offsets, key_offsets, n_sequences, tokens, key_tokens, n_heads, n_kv_heads, head_dim,
                                 causal, scale, head_dim <= 32 ? BwdShape<32>::kWalk : BwdShape<64>::kWalk);
    const BwdRows f{static_cast<const bf16 *>(output), static_cast<const bf16 *>(output_low),
                    static_cast<const bf16 *>(grad_output), grad_token_stride, grad_head_stride, lse, grad_lse,
                    static_cast<float *>(workspace)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    bf16 *dq = static_cast<bf16 *>(grad_query), *dk = static_cast<bf16 *>(grad_key),
         *dv = static_cast<bf16 *>(grad_value);
    switch (padded_dim(head_dim)) {
        case 32: return launch_backward<32>(A, q, k, v, g, f, dq, dk, dv, s);
        case 64: return launch_backward<64>(A, q, k, v, g, f, dq, dk, dv, s);
        default: return launch_backward<128>(A, q, k, v, g, f, dq, dk, dv, s);
    }
}
