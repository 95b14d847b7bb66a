// Calls the packed attention's and rotary's XLA handlers with buffers that fit one another, and with each of them in
// turn of another size or type.  The library's entry points are replaced by ones that only count: no handler may
// reach them with a buffer that they would read or write past its end.  Prints a line for each call.
#define rfdetr_packed_attention counted_attention
#define rfdetr_packed_attention_backward counted_attention_backward
#define rfdetr_axial_rotary counted_rotary
#include "../../rf-detr-jax_b200/ffi/rfdetr_ffi.cc"

#include <cstdio>
#include <functional>

static int calls = 0;

extern "C" int counted_attention(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t, const void *,
                                 int64_t, int64_t, const int32_t *, const int32_t *, void *, void *, float *, void *,
                                 size_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int, float) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_attention_backward(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t,
                                          const void *, int64_t, int64_t, const int32_t *, const int32_t *,
                                          const void *, const void *, const float *, const void *, int64_t, int64_t,
                                          const float *, void *, void *, void *, void *, size_t, int64_t, int64_t,
                                          int64_t, int64_t, int64_t, int64_t, int, float) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_rotary(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t, int, const void *,
                              int, const float *, const int64_t *, int64_t, void *, void *, int64_t, int64_t, int64_t,
                              int64_t, int, int) {
    return ++calls, RFDETR_OK;
}

using Dims = std::vector<int64_t>;

static void report(const char *name, const std::string &what, ffi::Error error) {
    std::printf("%s|%s|%s|%d\n", name, what.c_str(),
                error.code() == ffi::ErrorCode::kOk                ? "ok"
                : error.code() == ffi::ErrorCode::kInvalidArgument ? "refused"
                                                                   : "other",
                calls);
    calls = 0;
}

static std::string text(const Dims &d) {
    std::string s;
    for (int64_t x : d) s += (s.empty() ? "" : "x") + std::to_string(x);
    return "[" + s + "]";
}

// Calls `run` with the shapes as they are, and with each of them replaced in turn.
static void each(const char *name, const std::vector<Dims> &fit, const std::vector<std::vector<Dims>> &others,
                 const std::function<ffi::Error(const std::vector<Dims> &)> &run) {
    report(name, "fit", run(fit));
    for (size_t i = 0; i < fit.size(); ++i)
        for (const Dims &other : others[i]) {
            std::vector<Dims> d = fit;
            d[i] = other;
            report(name, std::to_string(i) + " " + text(other), run(d));
        }
}

int main() {
    using F = ffi::Buffer<ffi::F32>;
    using B = ffi::Buffer<ffi::BF16>;
    using I = ffi::Buffer<ffi::S32>;
    // 10 tokens of 4 heads over 7 of 2, 64 channels, 3 sequences.
    const Dims q{10, 4, 64}, k{7, 2, 64}, off{4}, lse{4, 10};
    const std::vector<Dims> like_q{{9, 4, 64}, {10, 3, 64}, {10, 4, 32}, {10, 256}}, like_lse{{4, 9}, {3, 10}, {40}};
    const std::vector<Dims> bad_q{{10, 4, 32}, {10, 256}}, bad_k{{7, 2, 32}, {6, 2, 64}, {7, 128}},
        bad_v{{6, 2, 64}, {7, 1, 64}, {7, 2, 32}, {7, 128}}, bad_off{{3}, {5}, {2, 2}, {}, {0}};
    each("attention", {q, k, k, off, off, q, q, lse},
         {bad_q, bad_k, bad_v, bad_off, bad_off, like_q, like_q, like_lse}, [](const std::vector<Dims> &d) {
             return (*RfdetrPackedAttention)(nullptr, {}, B(d[0]), B(d[1]), B(d[2]), I(d[3]), I(d[4]), 0, 0.125f,
                                             B(d[5]), B(d[6]), F(d[7]));
         });
    each("attention, no rest", {q, k, k, off, off, q, {0, 4, 64}, lse}, {{}, {}, {}, {}, {}, {}, {}, {}},
         [](const std::vector<Dims> &d) {
             return (*RfdetrPackedAttention)(nullptr, {}, B(d[0]), B(d[1]), B(d[2]), I(d[3]), I(d[4]), 0, 0.125f,
                                             B(d[5]), B(d[6]), F(d[7]));
         });
    each("backward", {q, k, k, off, off, q, q, lse, q, lse, q, k, k},
         {bad_q, bad_k, bad_v, bad_off, bad_off, like_q, {{0, 4, 64}, {9, 4, 64}, {10, 256}}, like_lse, like_q,
          like_lse, like_q, bad_v, bad_v},
         [](const std::vector<Dims> &d) {
             return (*RfdetrPackedAttentionBwd)(nullptr, {}, B(d[0]), B(d[1]), B(d[2]), I(d[3]), I(d[4]), B(d[5]),
                                                B(d[6]), F(d[7]), B(d[8]), F(d[9]), 0, 0.125f, B(d[10]), B(d[11]),
                                                B(d[12]));
         });
    // 10 tokens, 3 axes with 2 + 1 + 2 frequencies.
    using A = ffi::AnyBuffer;
    using T = ffi::DataType;
    const std::vector<int64_t> sections{2, 1, 2};
    const Dims rq{10, 4, 16}, rk{10, 2, 16};
    const std::vector<Dims> bad_rk{{9, 2, 16}, {10, 2, 8}, {10, 32}};
    auto rotary = [&](const std::vector<Dims> &d, T tq, T tk, T tp, T oq, T ok) {
        return (*RfdetrAxialRotary)(nullptr, A(tq, d[0]), A(tk, d[1]), A(tp, d[2]), F(d[3]), sections, 0, 0,
                                    A(oq, d[4]), A(ok, d[5]));
    };
    each("rotary", {rq, rk, {10, 3}, {5}, rq, rk},
         {{{9, 4, 16}, {10, 4, 8}, {10, 64}, {11, 4, 16}}, bad_rk, {{9, 3}, {10, 2}, {30}}, {{4}, {6}, {5, 1}, {}},
          {{9, 4, 16}, {10, 3, 16}, {10, 64}}, {{9, 2, 16}, {10, 1, 16}, {10, 32}}},
         [&](const std::vector<Dims> &d) { return rotary(d, T::BF16, T::BF16, T::S32, T::BF16, T::BF16); });
    const std::vector<Dims> fit{rq, rk, {10, 3}, {5}, rq, rk};
    for (T p : {T::F32, T::S32, T::S64}) report("rotary types", "fit", rotary(fit, T::F32, T::F32, p, T::F32, T::F32));
    report("rotary types", "key", rotary(fit, T::F32, T::BF16, T::F32, T::F32, T::BF16));
    report("rotary types", "query", rotary(fit, T::BF16, T::F32, T::F32, T::BF16, T::F32));
    report("rotary types", "query out", rotary(fit, T::F32, T::F32, T::F32, T::BF16, T::F32));
    report("rotary types", "key out", rotary(fit, T::F32, T::F32, T::F32, T::F32, T::BF16));
    report("rotary types", "positions", rotary(fit, T::F32, T::F32, T::BF16, T::F32, T::F32));
    report("rotary types", "positions", rotary(fit, T::F32, T::F32, T::F64, T::F32, T::F32));
    return 0;
}
