// A stand-in for the part of the XLA FFI header that rfdetr_ffi.cc uses, for compiling and calling its handlers
// where jaxlib is absent: buffers are shapes, types and addresses that a test makes up.  A handler is the function
// itself, and its binding is checked against the function's parameters.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <optional>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

namespace xla::ffi {

enum class DataType { U8, S32, S64, F16, BF16, F32, F64 };
inline constexpr DataType U8 = DataType::U8, S32 = DataType::S32, BF16 = DataType::BF16, F32 = DataType::F32;

inline size_t ByteWidth(DataType t) {
    return t == DataType::U8 ? 1
           : t == DataType::BF16 || t == DataType::F16 ? 2
           : t == DataType::S64 || t == DataType::F64 ? 8
                                                      : 4;
}

template <typename T>
class Span {
public:
    Span(const std::vector<std::remove_const_t<T>> &v) : data_(v.data()), size_(v.size()) {}
    T *begin() const { return data_; }
    T *end() const { return data_ + size_; }
    size_t size() const { return size_; }
    T &operator[](size_t i) const { return data_[i]; }

private:
    T *data_;
    size_t size_;
};

class AnyBuffer {
public:
    AnyBuffer(DataType type, std::vector<int64_t> dims, void *data = nullptr)
        : type_(type), dims_(std::move(dims)), data_(data) {}
    DataType element_type() const { return type_; }
    Span<const int64_t> dimensions() const { return dims_; }
    void *untyped_data() const { return data_; }
    size_t element_count() const {
        size_t n = 1;
        for (int64_t d : dims_) n *= static_cast<size_t>(d);
        return n;
    }

private:
    DataType type_;
    std::vector<int64_t> dims_;
    void *data_;
};

template <DataType> struct Native;
template <> struct Native<DataType::U8> { using T = uint8_t; };
template <> struct Native<DataType::S32> { using T = int32_t; };
template <> struct Native<DataType::BF16> { using T = uint16_t; };
template <> struct Native<DataType::F32> { using T = float; };

template <DataType D>
class Buffer : public AnyBuffer {
public:
    Buffer(std::vector<int64_t> dims, void *data = nullptr) : AnyBuffer(D, std::move(dims), data) {}
    typename Native<D>::T *typed_data() const { return static_cast<typename Native<D>::T *>(untyped_data()); }
};

template <typename T>
class Result {
public:
    Result(T value) : value_(std::move(value)) {}
    T &operator*() { return value_; }
    T *operator->() { return &value_; }

private:
    T value_;
};

enum class ErrorCode { kOk, kInvalidArgument, kInternal, kResourceExhausted };

class Error {
public:
    Error(ErrorCode code, std::string message) : code_(code), message_(std::move(message)) {}
    static Error Success() { return Error(ErrorCode::kOk, ""); }
    ErrorCode code() const { return code_; }

private:
    ErrorCode code_;
    std::string message_;
};

class ScratchAllocator {
public:
    std::optional<void *> Allocate(size_t, size_t = 1) { return reinterpret_cast<void *>(256); }
};

template <typename T> struct PlatformStream {};
template <typename T> struct CtxType { using Type = T; };
template <typename T> struct CtxType<PlatformStream<T>> { using Type = T; };

template <typename... P>
struct Binding {
    using Function = Error(P...);
    template <typename T> constexpr Binding<P..., typename CtxType<T>::Type> Ctx() const { return {}; }
    template <typename T> constexpr Binding<P..., T> Arg() const { return {}; }
    template <typename T> constexpr Binding<P..., T> Attr(const char *) const { return {}; }
    template <typename T> constexpr Binding<P..., Result<T>> Ret() const { return {}; }
};

struct Ffi {
    static constexpr Binding<> Bind() { return {}; }
};

}  // namespace xla::ffi

#define XLA_FFI_DEFINE_HANDLER_SYMBOL(symbol, function, ...)                                          \
    static_assert(std::is_same_v<decltype(__VA_ARGS__)::Function, std::remove_pointer_t<decltype(&function)>>); \
    [[maybe_unused]] static auto *const symbol = &function
