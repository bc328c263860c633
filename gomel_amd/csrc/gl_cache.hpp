// gl_cache.hpp -- the spectrogram cache and dropout (gl_cache.hip) as the handle's code (gomel_hip.hip) sees them, and the other way
// round.  Contract of the entry points: include/gomel_hip.h.
#pragma once
#include <hip/hip_runtime.h>

#include "gomel_host.hpp"

#define GL_HIDDEN __attribute__((visibility("hidden")))

struct gomel_cache {
    CacheLayout l;
    int device = 0;
    size_t n_slots = 0;
    uint8_t* store = nullptr;           // [n_slots][row_bytes]; the next two lie behind it in the same allocation
    int32_t* claim = nullptr;           // [n_slots], -1 between calls: which frame of a large write gets the slot
    unsigned long long* bad = nullptr;  // frames skipped because their slot was >= n_slots, since the cache was made
    std::mutex mu;                      // what is below
    unsigned long long told = 0;        // of them, reported by gomel_cache_bad_slots
    void* stage = nullptr;
    size_t stage_bytes = 0;
};

// defined in gl_cache.hip: device-side halves for callers that hold device pointers already.  `n` <= kMaxRows, arguments checked.
GL_HIDDEN hipError_t cache_write_device(gomel_cache* c, int type, const void* x, size_t xs, size_t n, const int64_t* slots, size_t first, void* y, size_t ys, hipStream_t s);
// strict: negative slots count as bad too; `bad` receives the count instead of the cache's counter
GL_HIDDEN hipError_t cache_read_device(gomel_cache* c, int type, void* y, size_t ys, size_t n, const int64_t* slots, size_t first, const DropRule& drop,
                                       uint64_t seed, uint64_t offset, bool strict, unsigned long long* bad, hipStream_t s);
// what kind of memory p is: 1 = memory of `device`, 0 = host memory, -1 = memory of another device
GL_HIDDEN int memory_kind(const void* p, int device);
// whether s is being captured into a graph
GL_HIDDEN bool stream_capturing(hipStream_t s);

// defined in gomel_hip.hip
// gomel_last_hip_error's value, by a function: a thread_local variable that another file declares is reached through its initialiser's
// address, which a hidden one without an initialiser has none of
GL_HIDDEN void set_last_hip(int e);
GL_HIDDEN int handle_device(const gomel_handle* h);
GL_HIDDEN int handle_num_mels(const gomel_handle* h);
GL_HIDDEN hipStream_t handle_stream(const gomel_handle* h);
GL_HIDDEN hipError_t handle_stage(gomel_handle* h, size_t bytes, void** p);   // from the handle's buffer pool
GL_HIDDEN void handle_unstage(gomel_handle* h, void* p);
