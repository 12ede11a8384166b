// Library-owned scratch buffers of the attention entry points that are called
// without a caller workspace (decode stream partials and arrival counters,
// decode split-K partials, prefill KV-split partials, the partials of the
// cascade decode over a shared prefix and of the shape-general kernels).
//
// One buffer per (device, stream, role), so calls on different streams never
// share memory.  Two rules make the buffers safe under hipGraph capture:
//   * A buffer that has been handed out is never freed.  A graph captured on
//     the stream keeps the buffer's address in its kernel arguments, so when a
//     later eager call needs more bytes the old buffer is retired (kept until
//     the process ends) and a new one of at least twice the size is
//     allocated; retired memory therefore stays below the live buffer's size.
//   * Nothing is allocated, cleared or synchronised while the stream is being
//     captured: get() then returns nullptr and the caller takes a path that
//     needs no scratch.
// A new buffer is cleared with an asynchronous memset on the caller's stream
// (ordered before the kernel that reads it); no host synchronisation.
//
// Host threads that share a stream share its buffers.  One launch alone is
// ordered by the stream; a call whose second launch reads what its first one
// left (partials, then their merge) keeps the buffer's WorkspaceHold until both
// are queued, so no other thread's launches come between them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>
#include <vector>

namespace rllm {

enum WorkspaceRole : int { WS_DECODE_STREAM = 0, WS_DECODE_PARTS = 1, WS_PREFILL_SPLITS = 2, WS_DECODE_PREFIX = 3, WS_GENERIC = 4,
                           WS_MX4_DECODE = 5, WS_MX4_PREFILL = 6, WS_SELECT = 7, WS_SPARSE = 8 };

// The sole right to queue launches on one buffer, until it is destroyed.
using WorkspaceHold = std::unique_lock<std::mutex>;

class WorkspaceCache {
public:
    // *out = a buffer of at least `bytes` for (current device, stream, role),
    // or nullptr when it would have to grow while the stream is capturing.
    // With `hold`, a buffer that is handed out is held by it.
    int32_t get(uintptr_t stream, int role, int64_t bytes, bool zero_new, void** out, WorkspaceHold* hold = nullptr) {
        *out = nullptr;
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess) return (int32_t)e;
        Entry* found;
        {
            std::lock_guard<std::mutex> lk(mu_);
            found = &live_[std::make_tuple(dev, stream, role)];   // entries are never moved or erased
        }
        Entry& ent = *found;
        WorkspaceHold lk(ent.queueing);   // mu_ is free: a held buffer keeps no other caller waiting
        if (ent.bytes >= bytes) {
            *out = ent.ptr;
            if (hold) *hold = std::move(lk);
            return 0;
        }
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        e = hipStreamIsCapturing(reinterpret_cast<hipStream_t>(stream), &cap);
        if (e != hipSuccess) return (int32_t)e;
        if (cap != hipStreamCaptureStatusNone) return 0;
        int64_t want = bytes > 2 * ent.bytes ? bytes : 2 * ent.bytes;
        want = (want + (1 << 20) - 1) & ~int64_t((1 << 20) - 1);
        void* p = nullptr;
        e = hipMalloc(&p, static_cast<size_t>(want));
        if (e != hipSuccess) return (int32_t)e;
        if (zero_new) {
            e = hipMemsetAsync(p, 0, static_cast<size_t>(want), reinterpret_cast<hipStream_t>(stream));
            if (e != hipSuccess) {
                retire(p);   // never freed once a queued operation may name it
                return (int32_t)e;
            }
        }
        if (ent.ptr) retire(ent.ptr);
        ent.ptr = p;
        ent.bytes = want;
        *out = p;
        if (hold) *hold = std::move(lk);
        return 0;
    }

private:
    struct Entry {
        std::mutex queueing;   // also guards the two below
        void* ptr = nullptr;
        int64_t bytes = 0;
    };
    void retire(void* p) {
        std::lock_guard<std::mutex> lk(mu_);
        retired_.push_back(p);
    }
    std::mutex mu_;   // guards the map and the list
    std::map<std::tuple<int, uintptr_t, int>, Entry> live_;
    std::vector<void*> retired_;
};

// one cache for the whole library (C++17 inline variable: a single instance
// across translation units)
inline WorkspaceCache g_workspaces;

}  // namespace rllm
