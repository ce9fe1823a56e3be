// A stand-in for the XLA FFI header, which ships with jax: the few names that the handlers use, with buffers that a test makes up. It lets
// them be compiled and called without jax; it says nothing of the real header's binding or calling convention.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

namespace xla::ffi {

enum class ErrorCode { kOk, kInternal, kInvalidArgument };
struct Error {
    ErrorCode code;
    std::string message;
    Error(ErrorCode c, std::string m) : code(c), message(std::move(m)) {}
    static Error Success() {
        return Error(ErrorCode::kOk, "");
    }
};
template <class T>
struct Span {
    std::vector<T> v;
    size_t size() const {
        return v.size();
    }
    const T* begin() const {
        return v.data();
    }
    const T* end() const {
        return v.data() + v.size();
    }
    const T& operator[](size_t i) const {
        return v[i];
    }
};
enum class DataType { BF16, F16, F32, F64, F8E4M3FN, S8, U8, S32, S64 };
struct AnyBuffer {
    void* data = nullptr;
    DataType type = DataType::F32;
    std::vector<int64_t> dims;
    void* untyped_data() const {
        return data;
    }
    DataType element_type() const {
        return type;
    }
    Span<const int64_t> dimensions() const;
    size_t element_count() const {
        size_t n = 1;
        for (int64_t d : dims) {
            n *= size_t(d);
        }
        return n;
    }
    size_t size_bytes() const {
        switch (type) {
        case DataType::F8E4M3FN:
        case DataType::S8:
        case DataType::U8: return element_count();
        case DataType::BF16:
        case DataType::F16: return 2 * element_count();
        case DataType::F64:
        case DataType::S64: return 8 * element_count();
        default: return 4 * element_count();
        }
    }
};
template <>
struct Span<const int64_t> : Span<int64_t> {
    Span(std::vector<int64_t> x = {}) : Span<int64_t>{std::move(x)} {}
};
inline Span<const int64_t> AnyBuffer::dimensions() const {
    return {dims};
}
template <class T>
struct Result {
    T t;
    T* operator->() {
        return &t;
    }
    T& operator*() {
        return t;
    }
};
template <class T>
struct ErrorOr {
    T t;
    bool has_error() const {
        return false;
    }
    Error error() const {
        return Error::Success();
    }
    T* operator->() {
        return &t;
    }
};
struct RemainingArgs {
    std::vector<AnyBuffer> v;
    size_t size() const {
        return v.size();
    }
    template <class T>
    ErrorOr<T> get(size_t i) const {
        return {v[i]};
    }
};
template <class T>
struct PlatformStream {};
enum class Traits { kCmdBufferCompatible };
struct Binder {
    template <class T>
    Binder Ctx() {
        return *this;
    }
    template <class T>
    Binder Arg() {
        return *this;
    }
    template <class T>
    Binder Ret() {
        return *this;
    }
    template <class T>
    Binder Attr(const char*) {
        return *this;
    }
    Binder RemainingArgs() {
        return *this;
    }
};
struct Ffi {
    static Binder Bind() {
        return {};
    }
};

} // namespace xla::ffi

#define XLA_FFI_DEFINE_HANDLER_SYMBOL(name, fn, binding, ...) \
    void* handler_##name() {                                  \
        (void)(binding);                                      \
        return reinterpret_cast<void*>(fn);                   \
    }
