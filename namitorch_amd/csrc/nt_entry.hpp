// nt_entry.hpp — argument checks and workspaces that the operators' entry points share.
#pragma once

#include <stdint.h>

#include <initializer_list>
#include <string>

#include "nt_internal.hpp"
#include "nt_pool.hpp"

namespace nt {

inline bool half_or_float(int32_t dtype) { return dtype == NT_F32 || dtype == NT_F16 || dtype == NT_BF16; }

// One array argument: `count` elements of `dtype` (or kInt32, kInt64), written or only read.
constexpr int32_t kInt32 = 100, kInt64 = 101;
struct Array {
    const void *ptr;
    int32_t dtype;
    uint64_t count;
    bool written, needed;
    uint64_t size() const { return dtype == NT_F32 || dtype == kInt32 ? 4u : dtype == kInt64 ? 8u : 2u; }
};

// Needed arrays are there, all are aligned to their dtype, and what is
// written overlaps nothing else.
inline int32_t check_arrays(const char *entry, std::initializer_list<Array> arrays) {
    for (const Array &a : arrays) {
        const uint64_t size = a.size();
        if (a.ptr == nullptr) {
            if (a.needed) return fail(NT_ERR_VALUE, std::string(entry) + ": NULL array");
            continue;
        }
        const uintptr_t start = (uintptr_t)a.ptr;
        if (start % size != 0) return fail(NT_ERR_VALUE, std::string(entry) + ": an array is not aligned to its dtype");
        if (!a.written) continue;
        for (const Array &b : arrays) {
            if (&a == &b || b.ptr == nullptr) continue;
            const uintptr_t other = (uintptr_t)b.ptr;
            if (start < other + b.count * b.size() && other < start + a.count * size)
                return fail(NT_ERR_VALUE, std::string(entry) + ": an output overlaps another array");
        }
    }
    return NT_OK;
}

// NT_ERR_RUNTIME while `stream` is captured: a replay would repeat a mask, or
// use a workspace that the pool has handed to others since.
inline int32_t refuse_capture(const char *entry, void *stream) {
    int32_t capturing = 0;
    const int32_t rc = nt_stream_capturing(stream, &capturing);
    if (rc != NT_OK) return rc;
    return capturing ? fail(NT_ERR_RUNTIME, std::string(entry) + ": not supported in stream capture") : NT_OK;
}

// Memory of the pool for one call, in parts; goes back as soon as the kernels
// are queued (the pool reuses it on this stream only).
class Workspace {
  public:
    template <class V>
    void want(V **at, uint64_t count) {
        entries_[used_++] = {reinterpret_cast<void **>(at), bytes_};
        bytes_ += (count * sizeof(V) + 255u) & ~255ull;
    }
    int32_t allocate(int32_t device, void *stream) {
        std::string error;
        const int32_t rc = device_pool().allocate(device, bytes_ > 0 ? bytes_ : 256u, stream, &base_, error);
        if (rc != NT_OK) return fail(rc, error);
        for (int k = 0; k < used_; ++k) *entries_[k].at = static_cast<char *>(base_) + entries_[k].offset;
        return NT_OK;
    }
    ~Workspace() {
        std::string error;
        if (base_ != nullptr) (void)device_pool().release(base_, error);
    }

  private:
    struct Entry {
        void **at;
        uint64_t offset;
    };
    Entry entries_[16];
    int used_ = 0;
    uint64_t bytes_ = 0;
    void *base_ = nullptr;
};

}  // namespace nt
