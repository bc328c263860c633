// gl_cache.hip -- the spectrogram cache (frames quantised as they are written, read back dequantised) and dropout from a
// counter-based generator: kernels, launches and the C ABI's entry points (include/gomel_hip.h holds the formulas and the contract).
// A translation unit of its own: nothing here shares device code with the Griffin-Lim kernels, and it is compiled without packed
// fp32 instructions (gomel_amd/build.py).
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "gl_cache.hpp"

#define GL_DEV static __device__ __forceinline__

namespace {

// ------------------------------------------------------------------------------------------------ element types
// In memory T, in registers W: fp32 for everything but fp64.  The one rounding to T is the hardware's round-to-nearest-even.  For fp16 the
// fp32 value is pinned first: the compiler would otherwise fold the multiply-add before it into a mixed-precision one with a single
// rounding in some kernels and not in others, and a value handed back by a write has to be, bit for bit, the value a read returns.
template <class T> struct Wide { typedef float type; };
template <> struct Wide<double> { typedef double type; };
GL_DEV float widen(float v) { return v; }
GL_DEV double widen(double v) { return v; }
GL_DEV float widen(__half v) { return __half2float(v); }
GL_DEV float widen(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class T> struct Narrow;
template <> struct Narrow<float> { GL_DEV float of(float v) { return v; } };
template <> struct Narrow<double> { GL_DEV double of(double v) { return v; } };
template <> struct Narrow<__half> { GL_DEV __half of(float v) { asm("" : "+v"(v)); return __float2half(v); } };
template <> struct Narrow<__hip_bfloat16> { GL_DEV __hip_bfloat16 of(float v) { return __float2bfloat16(v); } };
template <class T> GL_DEV T narrow(typename Wide<T>::type v) { return Narrow<T>::of(v); }

// ------------------------------------------------------------------------------------------------ the quantiser of one group
struct Scale { float lo, step; };

// A finite value as fp32, the largest fp32 number standing in for what lies beyond.
GL_DEV float to_f32(double v) { return fminf(fmaxf((float)v, -__FLT_MAX__), __FLT_MAX__); }

// mn, mx: extremes of the group's finite values (mn > mx: there are none); flags: 1 = a NaN, 2 = a +inf, 4 = a -inf among the others.
GL_DEV Scale group_scale(double mn, double mx, int flags, int levels) {
    if ((flags & 1) || (mn > mx && (flags & 6) == 6)) return Scale{__builtin_nanf(""), 0.0f};
    if (mn > mx) return Scale{(flags & 2) ? __builtin_inff() : -__builtin_inff(), 0.0f};
    const float lo = to_f32(mn), hi = to_f32(mx);
    return Scale{lo, (float)(((double)hi - (double)lo) / (double)levels)};
}
// fp64 because neighbouring codes meet at borders that fp32 quotients step over: 1 value in 3e4 would get the other code.
GL_DEV int quantise(double v, Scale s, int levels) {
    if (!(s.step > 0.0f)) return 0;
    const double q = rint((v - (double)s.lo) / (double)s.step);
    return (int)fmin(fmax(q, 0.0), (double)levels);
}
GL_DEV float dequantise(int q, Scale s, float) { return fmaf((float)q, s.step, s.lo); }
GL_DEV double dequantise(int q, Scale s, double) { return fma((double)q, (double)s.step, (double)s.lo); }

// ------------------------------------------------------------------------------------------------ the generator
GL_DEV uint64_t splitmix(uint64_t seed, uint64_t i) {   // the word of x0's sample i (k_init_x)
    uint64_t z = seed + (i + 1) * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
GL_DEV bool dropped(const DropRule& r, uint64_t seed, uint64_t e) {
    const uint64_t w = splitmix(seed, e >> 1);
    return r.all || (uint32_t)((e & 1) ? w >> 32 : w) < r.below;
}

struct Slots {   // where frame r goes / comes from
    const int64_t* at;
    int64_t first, n_slots;
};
GL_DEV int64_t slot_of(const Slots& s, int64_t r) { return s.at ? s.at[r] : s.first + r; }

struct WriteArgs {
    const void* x; void* y;
    int64_t xs, ys, n;
    Slots slots;
    uint8_t* store;
    CacheLayout l;
    const int32_t* claim;
    unsigned long long* bad;
};
struct ReadArgs {
    void* y;
    int64_t ys, n;
    Slots slots;
    const uint8_t* store;
    CacheLayout l;
    DropRule drop;
    int32_t dropping, strict;
    uint64_t seed, offset;
    unsigned long long* bad;
};

// Which frame keeps a slot that a write names more than once: the last.  The rows of a call claim their slots with an atomic maximum
// of the row index, the write below keeps the row whose claim stands, and k_claim_clear puts the -1 back.
__global__ void k_claim(Slots s, int64_t n, int32_t* claim) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= n) return;
    const int64_t slot = slot_of(s, r);
    if (slot >= 0 && slot < s.n_slots) atomicMax(claim + slot, (int32_t)r);
}
__global__ void k_claim_clear(Slots s, int64_t n, int32_t* claim) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= n) return;
    const int64_t slot = slot_of(s, r);
    if (slot >= 0 && slot < s.n_slots) claim[slot] = -1;
}

// One wave per frame, group after group: extremes, then codes (the second reading of the group comes from the cache).
template <class T> __global__ __launch_bounds__(64) void k_write(WriteArgs a) {
    typedef typename Wide<T>::type W;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x, K = a.l.K, levels = (1 << a.l.bits) - 1;
    const int64_t slot = slot_of(a.slots, r);
    if (slot < 0 || slot >= a.slots.n_slots) {
        if (slot >= a.slots.n_slots && lane == 0) atomicAdd(a.bad, 1ull);
        return;
    }
    const bool keep = !a.claim || a.claim[slot] == (int32_t)r;
    const T* x = (const T*)a.x + r * a.xs;
    T* y = a.y ? (T*)a.y + r * a.ys : nullptr;
    uint8_t* row = a.store + slot * a.l.row_bytes;
    for (int g = 0; g < a.l.groups; g++) {
        const int b0 = g * a.l.group, b1 = min(K, b0 + a.l.group);
        double mn = __builtin_inf(), mx = -__builtin_inf();
        int flags = 0;
        for (int i = 2 * b0 + lane; i < 2 * b1; i += 64) {
            const double v = (double)widen(x[i]);
            if (v != v) flags |= 1;
            else if (v == __builtin_inf()) flags |= 2;
            else if (v == -__builtin_inf()) flags |= 4;
            else { mn = fmin(mn, v); mx = fmax(mx, v); }
        }
        for (int m = 1; m < 64; m <<= 1) {
            mn = fmin(mn, __shfl_xor(mn, m));
            mx = fmax(mx, __shfl_xor(mx, m));
            flags |= __shfl_xor(flags, m);
        }
        const Scale s = group_scale(mn, mx, flags, levels);
        if (keep && lane == 0) *(float2*)(row + a.l.scale_off + 8 * g) = make_float2(s.lo, s.step);
        for (int b = b0 + lane; b < b1; b += 64) {
            const int q0 = quantise((double)widen(x[2 * b]), s, levels), q1 = quantise((double)widen(x[2 * b + 1]), s, levels);
            if (keep) {
                if (a.l.bits == 8) { row[2 * b] = (uint8_t)q0; row[2 * b + 1] = (uint8_t)q1; }
                else row[b] = (uint8_t)(q0 | q1 << 4);
            }
            if (y) { y[2 * b] = narrow<T>(dequantise(q0, s, W(0))); y[2 * b + 1] = narrow<T>(dequantise(q1, s, W(0))); }
        }
    }
}

// One lane per band.
template <class T> __global__ __launch_bounds__(64) void k_read(ReadArgs a) {
    typedef typename Wide<T>::type W;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    const int64_t slot = slot_of(a.slots, r);
    if (slot < 0 || slot >= a.slots.n_slots) {
        if ((slot >= a.slots.n_slots || a.strict) && lane == 0) atomicAdd(a.bad, 1ull);
        return;
    }
    const uint8_t* row = a.store + slot * a.l.row_bytes;
    T* y = (T*)a.y + r * a.ys;
    for (int b = lane; b < a.l.K; b += 64) {
        const float2 f = *(const float2*)(row + a.l.scale_off + 8 * (b / a.l.group));
        const Scale s{f.x, f.y};
        const int q0 = a.l.bits == 8 ? row[2 * b] : row[b] & 15, q1 = a.l.bits == 8 ? row[2 * b + 1] : row[b] >> 4;
        W v0 = dequantise(q0, s, W(0)), v1 = dequantise(q1, s, W(0));
        if (a.dropping) {
            const uint64_t e = a.offset + (uint64_t)r * (2 * a.l.K) + 2 * b;
            v0 = dropped(a.drop, a.seed, e) ? W(0) : v0 * (W)a.drop.scale;
            v1 = dropped(a.drop, a.seed, e + 1) ? W(0) : v1 * (W)a.drop.scale;
        }
        y[2 * b] = narrow<T>(v0); y[2 * b + 1] = narrow<T>(v1);
    }
}

struct DropArgs {
    const void* x; void* y;
    int64_t xs, ys, rows, cols;
    DropRule drop;
    uint64_t seed, offset;
};
template <class T> __global__ __launch_bounds__(256) void k_dropout(DropArgs a) {
    typedef typename Wide<T>::type W;
    const int64_t total = a.rows * a.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / a.cols, k = i - r * a.cols;
        const W v = widen(((const T*)a.x)[r * a.xs + k]);
        ((T*)a.y)[r * a.ys + k] = narrow<T>(dropped(a.drop, a.seed, a.offset + (uint64_t)i) ? W(0) : v * (W)a.drop.scale);
    }
}

#define GL_TYPES(type, CALL)                                  \
    switch (type) {                                           \
        case GOMEL_F64: { typedef double T; CALL; } break;    \
        case GOMEL_F32: { typedef float T; CALL; } break;     \
        case GOMEL_F16: { typedef __half T; CALL; } break;    \
        default: { typedef __hip_bfloat16 T; CALL; } break;   \
    }
// launches report their own status: hipGetLastError could hand back somebody else's
template <class Args> hipError_t launch(void (*k)(Args), unsigned grid, unsigned block, hipStream_t s, Args& a) {
    void* p[] = {&a};
    return hipLaunchKernel((const void*)k, dim3(grid), dim3(block), p, 0, s);
}
hipError_t launch_claim(void (*k)(Slots, int64_t, int32_t*), Slots sl, int64_t n, int32_t* claim, hipStream_t s) {
    void* p[] = {&sl, &n, &claim};
    return hipLaunchKernel((const void*)k, dim3((unsigned)((n + 255) / 256)), dim3(256), p, 0, s);
}

struct OnDevice {   // the calling thread's device switched to `dev` and back
    int prev = -1;
    hipError_t err = hipSuccess;
    explicit OnDevice(int dev) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != dev) err = hipSetDevice(dev);
        else prev = -1;
    }
    ~OnDevice() { if (prev >= 0) (void)hipSetDevice(prev); }
};
int hip_failed(hipError_t e) { g_last_hip = (int)e; (void)hipGetLastError(); return GOMEL_ERR_HIP; }
#define CHK(expr) do { const hipError_t e_ = (expr); if (e_ != hipSuccess) return hip_failed(e_); } while (0)

bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (!s) return false;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) { (void)hipGetLastError(); return false; }
    return st != hipStreamCaptureStatusNone;
}

hipError_t dropout_device(int type, const void* x, size_t xs, void* y, size_t ys, size_t rows, size_t cols, const DropRule& d, uint64_t seed, uint64_t offset, hipStream_t s) {
    DropArgs a{x, y, (int64_t)xs, (int64_t)ys, (int64_t)rows, (int64_t)cols, d, seed, offset};
    const unsigned grid = (unsigned)std::min<size_t>((rows * cols + 255) / 256, 65536);
    hipError_t e = hipSuccess;
    GL_TYPES(type, e = launch(k_dropout<T>, grid, 256, s, a));
    return e;
}

constexpr size_t kStageBytes = (size_t)32 << 20;

// Rows between host memory (stride elements apart) and a dense device buffer
hipError_t rows_in(void* dev, const char* host, size_t stride, size_t rows, size_t cols, size_t esz, hipStream_t s) {
    if (stride == cols || rows == 1) return hipMemcpyAsync(dev, host, rows * cols * esz, hipMemcpyHostToDevice, s);
    return hipMemcpy2DAsync(dev, cols * esz, host, stride * esz, cols * esz, rows, hipMemcpyHostToDevice, s);
}
hipError_t rows_out(char* host, const void* dev, size_t stride, size_t rows, size_t cols, size_t esz, hipStream_t s) {
    if (stride == cols || rows == 1) return hipMemcpyAsync(host, dev, rows * cols * esz, hipMemcpyDeviceToHost, s);
    return hipMemcpy2DAsync(host, stride * esz, dev, cols * esz, cols * esz, rows, hipMemcpyDeviceToHost, s);
}

int cache_stage(gomel_cache* c, size_t bytes, char** p) {   // caller holds c->mu
    if (c->stage_bytes < bytes) {
        if (c->stage) { CHK(hipFree(c->stage)); c->stage = nullptr; c->stage_bytes = 0; }
        CHK(hipMalloc(&c->stage, bytes));
        c->stage_bytes = bytes;
    }
    *p = (char*)c->stage;
    return GOMEL_OK;
}
// host slots: every one padding or inside the cache
int check_slots(const int64_t* slots, size_t n, size_t n_slots, bool pad_ok) {
    for (size_t i = 0; i < n; i++)
        if ((slots[i] < 0 && !pad_ok) || (slots[i] >= 0 && (uint64_t)slots[i] >= n_slots)) return GOMEL_ERR_TABLE_RANGE;
    return GOMEL_OK;
}

// What write and read share: the arguments checked, memory classified, and -- where something is in host memory -- the frames taken
// through the staging buffer in pieces.  `in` (write only) and `out` (write: values, may be null) are rows `is` / `os` elements apart.
template <class Run>
int cache_call(gomel_cache* c, int type, const void* in, size_t is, void* out, size_t os, size_t n, const int64_t* slots, size_t first, hipStream_t s, Run run) {
    const size_t cols = 2 * (size_t)c->l.K, esz = (size_t)type_bytes(type);
    if (!esz) return GOMEL_ERR_BAD_CONFIG;
    if (n == 0) return GOMEL_OK;
    if (n > kMaxRows || (in && !rows_span(n, cols, is)) || (out && !rows_span(n, cols, os))) return GOMEL_ERR_BAD_LENGTH;
    if (!slots && (first > c->n_slots || n > c->n_slots - first)) return GOMEL_ERR_TABLE_RANGE;
    if (in && out && !rows_disjoint_or_same(in, is, out, os, n, cols, esz)) return GOMEL_ERR_BAD_CONFIG;
    OnDevice dev(c->device); CHK(dev.err);
    const int ki = in ? memory_kind(in, c->device) : 1, ko = out ? memory_kind(out, c->device) : 1, ks = slots ? memory_kind(slots, c->device) : 1;
    if (ki < 0 || ko < 0 || ks < 0) return GOMEL_ERR_BAD_CONFIG;
    if (ki && ko && ks) { CHK(run(in, is, out, os, n, slots, first)); return GOMEL_OK; }
    if (capturing(s)) return GOMEL_ERR_BAD_CONFIG;
    if (!ks) { const int rc = check_slots(slots, n, c->n_slots, true); if (rc) return rc; }
    std::lock_guard<std::mutex> lk(c->mu);
    const size_t row = cols * esz, piece = std::min(n, std::max<size_t>(1, kStageBytes / row));
    const size_t part = (piece * row + 255) & ~(size_t)255;
    char* st = nullptr;
    const int rc = cache_stage(c, 2 * part + piece * 8, &st);   // frames | values or frames read | slots
    if (rc) return rc;
    char *st_out = st + part, *st_slots = st + 2 * part;
    hipError_t e = hipSuccess;
    for (size_t r = 0; r < n && e == hipSuccess; r += piece) {
        const size_t m = std::min(piece, n - r);
        const char* from = in ? (const char*)in + r * is * esz : nullptr;
        char* to = out ? (char*)out + r * os * esz : nullptr;
        const int64_t* at = slots ? slots + r : nullptr;
        if (!ks) e = hipMemcpyAsync(st_slots, at, m * 8, hipMemcpyHostToDevice, s);
        if (!ki && e == hipSuccess) e = rows_in(st, from, is, m, cols, esz, s);
        if (!ko && slots && e == hipSuccess) e = rows_in(st_out, to, os, m, cols, esz, s);   // rows of padding come back as they were
        if (e == hipSuccess) e = run(ki ? from : st, ki ? is : cols, ko ? to : st_out, ko ? os : cols, m, ks ? at : (const int64_t*)st_slots, first + r);
        if (!ko && e == hipSuccess) e = rows_out(to, st_out, os, m, cols, esz, s);
    }
    const hipError_t e2 = hipStreamSynchronize(s);   // also on an error: the staging buffer is free again when the lock goes
    if (e != hipSuccess) return hip_failed(e);
    CHK(e2);
    return GOMEL_OK;
}

int cache_create(gomel_handle* h, size_t n_slots, int bits, int group_bands, gomel_cache** out) {
    if (!h || !out) return GOMEL_ERR_NULL;
    *out = nullptr;
    if (n_slots == 0) return GOMEL_ERR_EMPTY;
    CacheLayout l;
    if (!cache_layout(handle_num_mels(h), bits, group_bands, &l) || n_slots > kMaxElems / (size_t)l.row_bytes) return GOMEL_ERR_BAD_CONFIG;
    gomel_cache* c = new (std::nothrow) gomel_cache();
    if (!c) return GOMEL_ERR_NO_MEMORY;
    c->l = l; c->device = handle_device(h); c->n_slots = n_slots;
    OnDevice dev(c->device);
    hipError_t e = dev.err;
    const size_t bytes = n_slots * (size_t)l.row_bytes;
    if (e == hipSuccess) e = hipMalloc((void**)&c->store, bytes);
    if (e == hipSuccess) e = hipMalloc((void**)&c->claim, n_slots * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&c->bad, 8);
    hipStream_t s = nullptr;   // its own: the default stream would wait for everybody's work
    if (e == hipSuccess) e = hipStreamCreateWithFlags(&s, hipStreamNonBlocking);
    if (e == hipSuccess) e = hipMemsetAsync(c->store, 0, bytes, s);
    if (e == hipSuccess) e = hipMemsetAsync(c->claim, 0xFF, n_slots * 4, s);
    if (e == hipSuccess) e = hipMemsetAsync(c->bad, 0, 8, s);
    if (s) {
        const hipError_t e2 = hipStreamSynchronize(s);
        if (e == hipSuccess) e = e2;
        (void)hipStreamDestroy(s);
    }
    if (e != hipSuccess) {
        if (c->store) (void)hipFree(c->store);
        if (c->claim) (void)hipFree(c->claim);
        if (c->bad) (void)hipFree(c->bad);
        delete c;
        return hip_failed(e);
    }
    *out = c;
    return GOMEL_OK;
}

int dropout_call(gomel_handle* h, int type, const void* x, size_t xs, void* y, size_t ys, size_t rows, size_t cols, double p, uint64_t seed, uint64_t offset, hipStream_t s) {
    if (!h) return GOMEL_ERR_NULL;
    const size_t esz = (size_t)type_bytes(type);
    DropRule d;
    if (!esz || !drop_rule(p, &d)) return GOMEL_ERR_BAD_CONFIG;
    if (rows == 0 || cols == 0) return GOMEL_OK;
    if (!x || !y) return GOMEL_ERR_NULL;
    if (!rows_span(rows, cols, xs) || !rows_span(rows, cols, ys)) return GOMEL_ERR_BAD_LENGTH;
    if (!rows_disjoint_or_same(x, xs, y, ys, rows, cols, esz)) return GOMEL_ERR_BAD_CONFIG;
    const int device = handle_device(h);
    OnDevice dev(device); CHK(dev.err);
    const int kx = memory_kind(x, device), ky = memory_kind(y, device);
    if (kx < 0 || ky < 0) return GOMEL_ERR_BAD_CONFIG;
    if (kx && ky) { CHK(dropout_device(type, x, xs, y, ys, rows, cols, d, seed, offset, s)); return GOMEL_OK; }
    if (capturing(s)) return GOMEL_ERR_BAD_CONFIG;
    // pieces of whole rows, or of one row where a row alone is larger than the staging buffer
    const size_t row = cols * esz, pr = std::max<size_t>(1, kStageBytes / row), pc = row > kStageBytes ? kStageBytes / esz : cols;
    const size_t bytes = std::min(rows, pr) * std::min(cols, pc) * esz;
    void* st = nullptr;
    CHK(handle_stage(h, bytes, &st));
    hipError_t e = hipSuccess;
    for (size_t r = 0; r < rows && e == hipSuccess; r += pr)
        for (size_t k = 0; k < cols && e == hipSuccess; k += pc) {
            const size_t m = std::min(pr, rows - r), w = std::min(pc, cols - k);
            const char* from = (const char*)x + (r * xs + k) * esz;
            char* to = (char*)y + (r * ys + k) * esz;
            if (!kx) e = rows_in(st, from, xs, m, w, esz, s);
            if (e == hipSuccess) e = dropout_device(type, kx ? from : st, kx ? xs : w, ky ? to : st, ky ? ys : w, m, w, d, seed, offset + r * cols + k, s);
            if (!ky && e == hipSuccess) e = rows_out(to, st, ys, m, w, esz, s);
        }
    const hipError_t e2 = hipStreamSynchronize(s);
    handle_unstage(h, st);
    if (e != hipSuccess) return hip_failed(e);
    CHK(e2);
    return GOMEL_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------------ device-side halves
int memory_kind(const void* p, int device) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) { (void)hipGetLastError(); return 0; }
    if (at.type == hipMemoryTypeDevice) return at.device == device ? 1 : -1;
    return 0;   // pageable, pinned and managed memory go through the staging buffer
}

hipError_t cache_write_device(gomel_cache* c, int type, const void* x, size_t xs, size_t n, const int64_t* slots, size_t first, void* y, size_t ys, hipStream_t s) {
    const bool claims = slots && n > 1;
    WriteArgs a{x, y, (int64_t)xs, (int64_t)ys, (int64_t)n, Slots{slots, (int64_t)first, (int64_t)c->n_slots}, c->store, c->l, claims ? c->claim : nullptr, c->bad};
    hipError_t e = hipSuccess;
    if (claims) e = launch_claim(k_claim, a.slots, a.n, c->claim, s);
    if (e == hipSuccess) GL_TYPES(type, e = launch(k_write<T>, (unsigned)n, 64, s, a));
    if (claims && e == hipSuccess) e = launch_claim(k_claim_clear, a.slots, a.n, c->claim, s);
    return e;
}

hipError_t cache_read_device(gomel_cache* c, int type, void* y, size_t ys, size_t n, const int64_t* slots, size_t first, const DropRule& drop,
                             uint64_t seed, uint64_t offset, bool strict, unsigned long long* bad, hipStream_t s) {
    ReadArgs a{y, (int64_t)ys, (int64_t)n, Slots{slots, (int64_t)first, (int64_t)c->n_slots}, c->store, c->l, drop, (int32_t)(drop.all || drop.below != 0),
               (int32_t)strict, seed, offset, bad ? bad : c->bad};
    hipError_t e = hipSuccess;
    GL_TYPES(type, e = launch(k_read<T>, (unsigned)n, 64, s, a));
    return e;
}

// ------------------------------------------------------------------------------------------------ C ABI
extern "C" {

int gomel_cache_create(gomel_handle* h, size_t n_slots, int bits, int group_bands, gomel_cache** out) {
    GOMEL_TRY return cache_create(h, n_slots, bits, group_bands, out); GOMEL_CATCH
}

int gomel_cache_destroy(gomel_cache* c) {
    if (!c) return GOMEL_OK;
    {
        OnDevice dev(c->device);
        hipError_t e = hipDeviceSynchronize();   // calls only queue work: it may still be running on any stream
        for (void* p : {(void*)c->store, (void*)c->claim, (void*)c->bad, c->stage}) {
            if (!p) continue;
            const hipError_t e2 = hipFree(p);
            if (e == hipSuccess) e = e2;
        }
        if (e != hipSuccess) { delete c; return hip_failed(e); }
    }
    delete c;
    return GOMEL_OK;
}

int gomel_cache_write(gomel_cache* c, int type, const void* frames, size_t stride, size_t n, const int64_t* slots, size_t first, void* values, size_t values_stride,
                      void* stream) {
    if (!c || (n && !frames)) return GOMEL_ERR_NULL;
    const hipStream_t s = (hipStream_t)stream;
    GOMEL_TRY
    return cache_call(c, type, frames, stride, values, values_stride, n, slots, first, s,
                      [&](const void* in, size_t is, void* out, size_t os, size_t m, const int64_t* at, size_t f) { return cache_write_device(c, type, in, is, m, at, f, out, os, s); });
    GOMEL_CATCH
}

int gomel_cache_read(gomel_cache* c, int type, void* frames, size_t stride, size_t n, const int64_t* slots, size_t first, double p, uint64_t seed, uint64_t offset,
                     void* stream) {
    if (!c || (n && !frames)) return GOMEL_ERR_NULL;
    DropRule d;
    if (!drop_rule(p, &d)) return GOMEL_ERR_BAD_CONFIG;
    const hipStream_t s = (hipStream_t)stream;
    const uint64_t cols = 2 * (uint64_t)c->l.K;
    GOMEL_TRY
    size_t done = 0;   // frames of earlier pieces: the counter of a piece's first element
    return cache_call(c, type, nullptr, 0, frames, stride, n, slots, first, s, [&](const void*, size_t, void* out, size_t os, size_t m, const int64_t* at, size_t f) {
        const hipError_t e = cache_read_device(c, type, out, os, m, at, f, d, seed, offset + done * cols, false, nullptr, s);
        done += m;
        return e;
    });
    GOMEL_CATCH
}

int gomel_cache_bad_slots(gomel_cache* c, uint64_t* count) {
    if (!c || !count) return GOMEL_ERR_NULL;
    OnDevice dev(c->device); CHK(dev.err);
    std::lock_guard<std::mutex> lk(c->mu);
    hipStream_t s = nullptr;
    CHK(hipStreamCreateWithFlags(&s, hipStreamNonBlocking));
    unsigned long long got = 0;
    hipError_t e = hipMemcpyAsync(&got, c->bad, 8, hipMemcpyDeviceToHost, s);
    if (e == hipSuccess) e = hipMemsetAsync(c->bad, 0, 8, s);
    const hipError_t e2 = hipStreamSynchronize(s);
    (void)hipStreamDestroy(s);
    if (e == hipSuccess) e = e2;
    if (e != hipSuccess) return hip_failed(e);
    *count = got;
    return GOMEL_OK;
}

int gomel_dropout(gomel_handle* h, int type, const void* x, size_t x_stride, void* y, size_t y_stride, size_t rows, size_t cols, double p, uint64_t seed, uint64_t offset,
                  void* stream) {
    GOMEL_TRY return dropout_call(h, type, x, x_stride, y, y_stride, rows, cols, p, seed, offset, (hipStream_t)stream); GOMEL_CATCH
}
int gomel_dropout_backward(gomel_handle* h, int type, const void* dy, size_t dy_stride, void* dx, size_t dx_stride, size_t rows, size_t cols, double p, uint64_t seed,
                           uint64_t offset, void* stream) {
    GOMEL_TRY return dropout_call(h, type, dy, dy_stride, dx, dx_stride, rows, cols, p, seed, offset, (hipStream_t)stream); GOMEL_CATCH
}

}  // extern "C"
