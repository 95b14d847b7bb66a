// Calls the XLA handlers of the changed scores, the normed rotary positions and the clipping with buffers that fit one
// another, and with each of them in turn of another size or type.  The library's entry points are replaced by ones that
// only count.  Prints a line for each call.
#define rfdetr_packed_attention_scored counted_scored
#define rfdetr_packed_attention_scored_backward counted_scored_backward
#define rfdetr_normed_rotary counted_normed
#define rfdetr_normed_rotary_backward counted_normed_backward
#define rfdetr_clip_gradients counted_clip
#include "../../rf-detr-jax_b200/ffi/rfdetr_ffi.cc"

#include <cstdio>
#include <functional>

static int calls = 0;

extern "C" int counted_scored(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t, const void *, int64_t,
                              int64_t, const int32_t *, const int32_t *, void *, void *, float *, void *, size_t, int64_t,
                              int64_t, int64_t, int64_t, int64_t, int64_t, int, float, float, const float *,
                              const int32_t *) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_scored_backward(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t,
                                       const void *, int64_t, int64_t, const int32_t *, const int32_t *, const void *,
                                       const void *, const float *, const void *, int64_t, int64_t, const float *, void *,
                                       void *, void *, void *, size_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                                       int64_t, int, float, float, const float *, const int32_t *) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_normed(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t, int, const void *, int,
                              const void *, int, float, const void *, int, const float *, const int64_t *, int64_t,
                              void *, void *, int64_t, int64_t, int64_t, int64_t, int) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_normed_backward(void *, const void *, int64_t, int64_t, const void *, int64_t, int64_t,
                                       const void *, int64_t, int64_t, const void *, int64_t, int64_t, int, const void *,
                                       int, const void *, int, float, const void *, int, const float *, const int64_t *,
                                       int64_t, void *, void *, void *, void *, void *, size_t, int64_t, int64_t, int64_t,
                                       int64_t, int) {
    return ++calls, RFDETR_OK;
}
extern "C" int counted_clip(void *, const void *const *, const int32_t *, void *const *, const int32_t *, const int64_t *,
                            int64_t, double, float *, void *, size_t) {
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

// Calls `run` with the shapes as they are, and with each of them replaced in turn.
static void each(const char *name, const std::vector<Dims> &fit, const std::vector<std::vector<Dims>> &others,
                 const std::function<ffi::Error(const std::vector<Dims> &)> &run) {
    report(name, "fit", run(fit));
    for (size_t i = 0; i < others.size(); ++i)
        for (const Dims &other : others[i]) {
            std::vector<Dims> d = fit;
            d[i] = other;
            report(name, std::to_string(i), run(d));
        }
}

int main() {
    using F = ffi::Buffer<ffi::F32>;
    using B = ffi::Buffer<ffi::BF16>;
    using I = ffi::Buffer<ffi::S32>;
    using A = ffi::AnyBuffer;
    using T = ffi::DataType;
    // 10 tokens of 4 heads over 7 of 2, 64 channels, 3 sequences.
    const Dims q{10, 4, 64}, k{7, 2, 64}, off{4}, lse{4, 10}, slopes{4}, prefix{3};
    const std::vector<Dims> bad_q{{10, 4, 32}, {10, 256}}, bad_k{{7, 2, 32}, {6, 2, 64}}, bad_v{{6, 2, 64}, {7, 1, 64}},
        bad_off{{3}, {2, 2}, {0}}, bad_m{{3}, {8}, {2, 2}}, bad_p{{2}, {4}, {}}, like_q{{9, 4, 64}, {10, 256}},
        like_lse{{4, 9}, {40}};
    for (const bool some : {true, false})
        each("scored", {q, k, k, off, off, some ? slopes : Dims{0}, some ? prefix : Dims{0}, q, q, lse},
             {bad_q, bad_k, bad_v, bad_off, bad_off, bad_m, bad_p, like_q, like_q, like_lse},
             [](const std::vector<Dims> &d) {
                 return (*RfdetrScoredAttention)(nullptr, {}, B(d[0]), B(d[1]), B(d[2]), I(d[3]), I(d[4]), F(d[5]),
                                                 I(d[6]), 1, 0.125f, 30.0f, B(d[7]), B(d[8]), F(d[9]));
             });
    each("scored backward", {q, k, k, off, off, slopes, prefix, q, q, lse, q, lse, q, k, k},
         {bad_q, bad_k, bad_v, bad_off, bad_off, bad_m, bad_p, like_q, like_q, like_lse, like_q, like_lse, like_q, bad_v,
          bad_v},
         [](const std::vector<Dims> &d) {
             return (*RfdetrScoredAttentionBwd)(nullptr, {}, B(d[0]), B(d[1]), B(d[2]), I(d[3]), I(d[4]), F(d[5]), I(d[6]),
                                                B(d[7]), B(d[8]), F(d[9]), B(d[10]), F(d[11]), 1, 0.125f, 30.0f, B(d[12]),
                                                B(d[13]), B(d[14]));
         });
    // 10 tokens, 3 axes with 2 + 1 + 2 frequencies, 16 channels.
    const std::vector<int64_t> sections{2, 1, 2};
    const Dims rq{10, 4, 16}, rk{10, 2, 16}, w{16}, pos{10, 3}, freq{5};
    const std::vector<Dims> bad_rq{{9, 4, 16}, {10, 64}}, bad_rk{{9, 2, 16}, {10, 2, 8}, {10, 32}}, bad_w{{8}, {4, 4}, {}},
        bad_pos{{9, 3}, {10, 2}}, bad_freq{{4}, {5, 1}}, like_rk{{10, 1, 16}, {9, 2, 16}, {320}};
    auto normed = [&](const std::vector<Dims> &d, T in, T wt, T pt, T out) {
        return (*RfdetrNormedRotary)(nullptr, A(in, d[0]), A(in, d[1]), A(wt, d[2]), A(wt, d[3]), A(pt, d[4]), F(d[5]),
                                     sections, 0, 1e-6f, A(out, d[6]), A(out, d[7]));
    };
    const std::vector<Dims> fit{rq, rk, w, w, pos, freq, rq, rk};
    each("normed", fit, {bad_rq, bad_rk, bad_w, bad_w, bad_pos, bad_freq, bad_rq, like_rk},
         [&](const std::vector<Dims> &d) { return normed(d, T::BF16, T::F32, T::S32, T::BF16); });
    report("normed, no weights", "fit", normed({rq, rk, {0}, {0}, pos, freq, rq, rk}, T::F32, T::F32, T::S64, T::F32));
    report("normed types", "positions", normed(fit, T::F32, T::F32, T::F64, T::F32));
    report("normed types", "out", normed(fit, T::F32, T::F32, T::F32, T::BF16));
    auto back = [&](const std::vector<Dims> &d, T in, T wt, T gt, T out, T dwt) {
        return (*RfdetrNormedRotaryBwd)(nullptr, {}, A(in, d[0]), A(in, d[1]), A(wt, d[2]), A(wt, d[3]), A(T::S32, d[4]),
                                        F(d[5]), A(gt, d[6]), A(gt, d[7]), sections, 0, 1e-6f, A(out, d[8]), A(out, d[9]),
                                        A(dwt, d[10]), A(dwt, d[11]));
    };
    const std::vector<Dims> fit_back{rq, rk, w, w, pos, freq, rq, rk, rq, rk, w, w};
    each("normed backward", fit_back,
         {bad_rq, bad_rk, bad_w, bad_w, bad_pos, bad_freq, bad_rq, like_rk, bad_rq, like_rk, {{8}, {0}}, {{8}, {0}}},
         [&](const std::vector<Dims> &d) { return back(d, T::F32, T::BF16, T::F32, T::F32, T::BF16); });
    report("normed backward types", "cotangent", back(fit_back, T::F32, T::F32, T::BF16, T::F32, T::F32));
    report("normed backward types", "gradient", back(fit_back, T::F32, T::F32, T::F32, T::BF16, T::F32));
    report("normed backward types", "weight", back(fit_back, T::F32, T::F32, T::F32, T::F32, T::BF16));
    each("clip", {{100}, {100}, {1}}, {{{99}, {10, 10}, {}}, {{99}, {101}}, {{2}, {}}}, [](const std::vector<Dims> &d) {
        return (*RfdetrClipGradients)(nullptr, {}, A(T::BF16, d[0]), 1.0f, A(T::F32, d[1]), F(d[2]));
    });
    return 0;
}
