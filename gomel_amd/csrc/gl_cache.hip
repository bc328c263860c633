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
GL_DEV float to_f32(float v) { return v; }
// mn, mx: extremes of the group's finite values (mn > mx: there are none); flags: 1 = a NaN, 2 = a +inf, 4 = a -inf among the others.
template <class W> GL_DEV Scale group_scale(W mn, W mx, int flags, int levels) {
    const bool none = mn > mx;
    if (flags & 1 || (none && (flags & 6) == 6)) return Scale{__builtin_nanf(""), 0.0f};
    if (none) return Scale{(flags & 2) ? __builtin_inff() : -__builtin_inff(), 0.0f};
    const float lo = to_f32(mn), hi = to_f32(mx);
    // the quotient by a constant, correctly rounded: the product with the rounded reciprocal, its remainder by multiply-add, one
    // correction (Markstein 1990); equal to the division on 4e8 pairs of fp32 numbers of every size
    const double d = (double)hi - (double)lo, over = levels == 255 ? 1.0 / 255.0 : 1.0 / 15.0, q = d * over;
    return Scale{lo, (float)fma(fma(-q, (double)levels, d), over, q)};
}
// The code of v as a number, rint((v - lo) / step) in fp64: neighbouring codes meet at borders that fp32 quotients step over (1 value in 3e4
// would get the other code).  NaN and infinities: fmaxf / fminf return the number.
GL_DEV float code_of(double v, Scale s, float levels) {
    if (!(s.step > 0.0f)) return 0.0f;
    return fminf(fmaxf((float)rint((v - (double)s.lo) / (double)s.step), 0.0f), levels);
}
// The codes of N values at once.  The quotients come from products with 1 / step first, and a value whose product is so near a border that
// the rounding of difference, reciprocal and product could have carried it across sends the lane to the definition.
//   fp32 (and the 16-bit types): v - lo is off by 2^-24 of itself, v_rcp_f32 by 2^-23, the product by 2^-24: 2^-22 of a quotient of at
// most `levels` (and a little), so levels * 2^-21 is twice what is needed; one value in 4000 is that near at 8 bits.  Instructions of
// either width cost the same here, but the definition takes twice as many: a write of 16-bit frames was bound by them (192 bands: 740
// vector instructions per wave and 193 us for 409 600 frames with values, now 489 and 159).
//   fp64: 2^-51 of the quotient; 2^-33 is far beyond it and as rare as never.
// Whatever is not a number in between (an infinite value, a step whose reciprocal fp32 does not hold) fails the comparison and goes there too.
template <int N> GL_DEV void quantise(const float* v, Scale s, float per, float levels, float* q) {
    const float limit = 0.5f - levels * 0x1p-21f;
    bool sure[N], all = true;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float t = (v[j] - s.lo) * per;
        q[j] = rintf(t);
        all &= sure[j] = fabsf(t - q[j]) <= limit;
    }
    if (!all) {   // value by value: 16-bit frames meet exact ties (one value in 500 at 8 bits), seldom two in a unit
#pragma unroll
        for (int j = 0; j < N; j++) if (!sure[j]) q[j] = code_of((double)v[j], s, levels);
    }
}
template <int N> GL_DEV void quantise(const double* v, Scale s, double per, float levels, float* q) {
    bool sure[N], all = true;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const double t = (v[j] - (double)s.lo) * per, r = rint(t);
        all &= sure[j] = fabs(t - r) <= 0.5 - 0x1p-33;
        q[j] = fminf(fmaxf((float)r, 0.0f), levels);
    }
    if (!all) {
#pragma unroll
        for (int j = 0; j < N; j++) if (!sure[j]) q[j] = code_of(v[j], s, levels);
    }
}
// 1 / step for them: 0 for step = 0 (all codes are 0), NaN where v_rcp_f32 would return 0 for a step whose reciprocal is subnormal.
GL_DEV float reciprocal(Scale s, float) { return s.step > 0.0f ? (s.step < 0x1p126f ? __builtin_amdgcn_rcpf(s.step) : __builtin_nanf("")) : 0.0f; }
GL_DEV double reciprocal(Scale s, double) { return s.step > 0.0f ? 1.0 / (double)s.step : 0.0; }
GL_DEV float dequantise(float q, Scale s, float) { return fmaf(q, s.step, s.lo); }
GL_DEV double dequantise(float q, Scale s, double) { return fma((double)q, (double)s.step, (double)s.lo); }

// ------------------------------------------------------------------------------------------------ the generator
constexpr uint64_t kGamma = 0x9E3779B97F4A7C15ull;
GL_DEV uint64_t splitmix_of(uint64_t z) {   // the word of x0's sample i (k_init_x): z = seed + (i + 1) * kGamma
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// ------------------------------------------------------------------------------------------------ 16-byte units
// A lane moves 16 bytes of frames or activations at a time: UV values of T.  Rows may start at any element (gfx950 takes a 16-byte access
// at any element's alignment), a row's last unit may be partial: its first value then stands in the places behind the row's end, where
// it changes no extreme.
template <class T> constexpr int UV = 16 / (int)sizeof(T);
typedef uint32_t raw_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t raw_word __attribute__((ext_vector_type(4), aligned(4)));
template <class T> struct Raw { typedef raw_word type; };
template <> struct Raw<__half> { typedef raw_any type; };
template <> struct Raw<__hip_bfloat16> { typedef raw_any type; };
template <class T> struct Unit {
    T v[UV<T>];
    template <bool S> static __device__ __forceinline__ Unit load(const T* p, int n) {
        Unit u;
        if (n >= UV<T>) {
            typename Raw<T>::type r;
            if (S) r = __builtin_nontemporal_load((const typename Raw<T>::type*)p);
            else r = *(const typename Raw<T>::type*)p;
            __builtin_memcpy(u.v, &r, 16);
        } else {
#pragma unroll
            for (int j = 0; j < UV<T>; j++) u.v[j] = p[j < n ? j : 0];   // n >= 1
        }
        return u;
    }
    template <bool S> __device__ __forceinline__ void store(T* p, int n) const {
        if (n >= UV<T>) {
            typename Raw<T>::type r;
            __builtin_memcpy(&r, v, 16);
            if (S) __builtin_nontemporal_store(r, (typename Raw<T>::type*)p);
            else *(typename Raw<T>::type*)p = r;
        } else {
#pragma unroll
            for (int j = 0; j < UV<T>; j++) if (j < n) p[j] = v[j];
        }
    }
};

// How a frame lies over a wave: in 2^lanes_log2 neighbouring lanes, `units` units each, `lanes` apart, so that every access of the wave is
// one run of memory and what depends on the frame alone (its slot, its addresses) is worked out once per lane.  A frame too wide for
// that is cut into `segs` segments of 64 lanes x 4 units (units = 0: k_write cannot, it needs the extremes of the whole frame).  Up to
// kSpreadRows frames a wave each fits the chip: then all 64 lanes, and the fewest units after each other (a write of 64 frames of 160
// bands in fp16: 5.6 us with 64 lanes x 1 unit, 8.6 with 8 x 5).
struct Spread { int32_t lanes_log2, units, segs; };
constexpr int kMostUnits = 6;
constexpr size_t kSpreadRows = 4096;
inline Spread spread_of(size_t n, int upr, int least_lanes_log2, bool may_cut) {
    Spread p{6, 0, 1};
    if (n <= kSpreadRows) least_lanes_log2 = 6;
    // the pair with the fewest idle places, the most lanes among equals
    for (int lg = 6, best = INT32_MAX; lg >= least_lanes_log2; lg--) {
        const int k = (upr + (1 << lg) - 1) >> lg;
        if (k <= kMostUnits && (k << lg) < best) { best = k << lg; p.units = k; p.lanes_log2 = lg; }
    }
    if (!p.units && may_cut) { p.units = 4; p.segs = (upr + 255) / 256; }
    return p;
}

// How a grid of blocks walks rows of `upr` units each, one unit per lane: short rows share a block (`rpb` rows of them), a long row is cut
// into `segs` segments (rpb = 0).  The block size is the multiple of a wave that leaves the fewest lanes without a unit.  The quotient
// i / upr of a unit's index in its block is exact for i, upr < 2^16.
struct Walk {
    int64_t rows, upr, segs, blocks;
    int32_t rpb, block;
    uint32_t magic;
};
inline Walk walk_of(size_t rows, size_t upr) {
    Walk w{(int64_t)rows, (int64_t)upr, 0, 0, 0, 256, 0};
    double best = 0;
    for (int block : {256, 192, 320, 384, 128, 448, 512, 64}) {
        const size_t b = (size_t)block, used = upr <= b ? b / upr * upr : upr, of = upr <= b ? b : (upr + b - 1) / b * b;
        const double share = (double)used / (double)of;
        if (share > best + 0.01) { best = share; w.block = block; }
    }
    const size_t b = (size_t)w.block;
    if (upr <= b) {
        w.rpb = (int32_t)(b / upr);
        w.magic = (uint32_t)(((uint64_t)1 << 32) / upr + 1);
        w.blocks = (int64_t)((rows + w.rpb - 1) / w.rpb);
    } else {
        w.segs = (int64_t)((upr + b - 1) / b);
        w.blocks = (int64_t)rows * w.segs;
    }
    return w;
}
GL_DEV bool walk_unit(const Walk& w, int64_t block, int64_t* r, int64_t* u) {   // this lane's unit; false: there is none
    const int i = (int)threadIdx.x;
    if (w.rpb) {
        const uint32_t q = w.upr == 1 ? (uint32_t)i : (uint32_t)(((uint64_t)(uint32_t)i * w.magic) >> 32);
        *r = block * w.rpb + q;
        *u = i - (int64_t)q * w.upr;
        return (int)q < w.rpb && *r < w.rows;
    }
    const int64_t b = block / w.segs;
    *r = b;
    *u = (block - b * w.segs) * w.block + i;
    return *u < w.upr;
}

// A claim is read past this compute unit's and this die's caches: a call on another stream may be claiming neighbouring slots (the same
// cache line) right now, and a line kept from before that would show this call's claims as they were then.  The -1 that takes a claim
// back is an ordinary store: it is written back, by its own bytes, before the next kernel of the stream starts.
GL_DEV int32_t claim_of(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

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
    int32_t* claim;           // null: a frame looks through the later slots of the call itself
    unsigned long long* bad;
    Spread p;
    int32_t gunits_log2;      // a group's units
    int64_t block0 = 0;
};
struct ReadArgs {
    void* y;
    int64_t ys, n;
    Slots slots;
    const uint8_t* store;
    CacheLayout l;
    Spread p;
    DropRule drop;
    int32_t gshift, strict;   // a band's group = band >> gshift
    uint64_t seed, offset;
    unsigned long long* bad;
    int32_t wraps;            // offset + the output's elements pass 2^64
    int64_t block0 = 0;
};

// Which frame keeps a slot that a write names more than once: the last.  The rows of a call claim their slots with an atomic maximum
// of the row index, the write below keeps the row whose claim stands and puts the -1 back (k_claim_clear does where several parts of the
// grid share a frame).  4.7 us for 102 400 slots, bound by the atomics' way to memory.
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

// Extremes of a group while they are being gathered.  fp32: gfx950's three-operand minimum and maximum, one instruction for two values, which
// hand a NaN on: what is not finite shows in the extremes themselves.  fp64: `odd` turns NaN.
GL_DEV float least(float a, float b) { asm("v_minimum3_f32 %0, %0, %1, %1" : "+v"(a) : "v"(b)); return a; }
GL_DEV float most(float a, float b) { asm("v_maximum3_f32 %0, %0, %1, %1" : "+v"(a) : "v"(b)); return a; }
GL_DEV double least(double a, double b) { return fmin(a, b); }
GL_DEV double most(double a, double b) { return fmax(a, b); }
// The value of another lane of the same 2 M neighbouring lanes, M being the power of two that was reached: the first M hold one value, the
// other M theirs, and each gets one of the other's.  Within 16 lanes a move through the vector unit's own crossbar, no trip to LDS.
template <int M> GL_DEV float other(float v) {
    const int i = __builtin_bit_cast(int, v);
    if (M == 1) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0xB1, 0xF, 0xF, false));    // quad_perm 1,0,3,2
    if (M == 2) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x4E, 0xF, 0xF, false));    // quad_perm 2,3,0,1
    if (M == 4) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x141, 0xF, 0xF, false));   // row_half_mirror
    if (M == 8) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x140, 0xF, 0xF, false));   // row_mirror
    return __shfl_xor(v, M);
}
template <int M> GL_DEV double other(double v) {
    if (M > 8) return __shfl_xor(v, M);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const float lo = other<M>(__builtin_bit_cast(float, (uint32_t)b)), hi = other<M>(__builtin_bit_cast(float, (uint32_t)(b >> 32)));
    return __builtin_bit_cast(double, (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo));
}
// Extremes over `span` neighbouring lanes (a power of two), in each of them.
template <class W> GL_DEV void join(int span, W* mn, W* mx) {
    if (span > 1) { *mn = least(*mn, other<1>(*mn)); *mx = most(*mx, other<1>(*mx)); }
    if (span > 2) { *mn = least(*mn, other<2>(*mn)); *mx = most(*mx, other<2>(*mx)); }
    if (span > 4) { *mn = least(*mn, other<4>(*mn)); *mx = most(*mx, other<4>(*mx)); }
    if (span > 8) { *mn = least(*mn, other<8>(*mn)); *mx = most(*mx, other<8>(*mx)); }
    if (span > 16) { *mn = least(*mn, other<16>(*mn)); *mx = most(*mx, other<16>(*mx)); }
    if (span > 32) { *mn = least(*mn, other<32>(*mn)); *mx = most(*mx, other<32>(*mx)); }
}
template <class W> struct Range;
template <> struct Range<float> {
    float mn = __builtin_inff(), mx = -__builtin_inff();
    __device__ __forceinline__ void add(float a, float b) {
        asm("v_minimum3_f32 %0, %0, %1, %2" : "+v"(mn) : "v"(a), "v"(b));
        asm("v_maximum3_f32 %0, %0, %1, %2" : "+v"(mx) : "v"(a), "v"(b));
    }
    // (a lane that has added nothing: mn = +inf, mx = -inf)
    __device__ __forceinline__ bool special() const { return !(mn > -__builtin_inff() && mx < __builtin_inff()); }
};
template <> struct Range<double> {
    double mn = __builtin_inf(), mx = -__builtin_inf(), odd = 0;
    __device__ __forceinline__ void add(double a, double b) {
        mn = fmin(mn, fmin(a, b));
        mx = fmax(mx, fmax(a, b));
        odd = fma(a, 0.0, fma(b, 0.0, odd));
    }
    __device__ __forceinline__ bool special() const { return !(odd == 0.0); }
};
// The same with the finite values only, and what the others are (group_scale's flags).
template <class W> GL_DEV void add_finite(W v, W* mn, W* mx, int* flags) {
    if (v != v) *flags |= 1;
    else if (v == (W)__builtin_inf()) *flags |= 2;
    else if (v == -(W)__builtin_inf()) *flags |= 4;
    else { *mn = least(*mn, v); *mx = most(*mx, v); }
}

template <int B, bool S> GL_DEV void put_code(uint8_t* p, const uint32_t* code) {   // B bytes, aligned to themselves
    if (B == 8) {
        typedef uint32_t two __attribute__((ext_vector_type(2)));
        const two v = {code[0], code[B == 8]};
        if (S) __builtin_nontemporal_store(v, (two*)p);
        else *(two*)p = v;
    } else if (B == 4) {
        if (S) __builtin_nontemporal_store(code[0], (uint32_t*)p);
        else *(uint32_t*)p = code[0];
    } else if (B == 2) {
        if (S) __builtin_nontemporal_store((uint16_t)code[0], (uint16_t*)p);
        else *(uint16_t*)p = (uint16_t)code[0];
    } else {
        if (S) __builtin_nontemporal_store((uint8_t)code[0], p);
        else *p = (uint8_t)code[0];
    }
}
// One unit's codes into the row and, when they are asked for, its values.  S: what is stored past the caches (kStreamBytes): 1 the values,
// 2 the codes as well.
template <class T, int S> GL_DEV void put_unit(const WriteArgs& a, uint8_t* row, T* y, bool keep, int u, int n, const typename Wide<T>::type* w, Scale s, typename Wide<T>::type per) {
    typedef typename Wide<T>::type W;
    const bool wide = a.l.bits == 8;
    const float levels = wide ? 255.0f : 15.0f;
    Unit<T> out;
    uint32_t code[2] = {0, 0};
    float q[UV<T>];
    quantise<UV<T>>(w, s, per, levels, q);
    if (keep) {
        if (wide) {
#pragma unroll
            for (int j = 0; j < UV<T>; j++) code[j / 4] = __builtin_amdgcn_cvt_pk_u8_f32(q[j], j % 4, code[j / 4]);
            put_code<UV<T>, (S > 1)>(row + u * UV<T>, code);
        } else {
#pragma unroll
            for (int j = 0; j < UV<T>; j += 4) {   // four codes make a number below 2^16, exact in fp32
                float four = q[j] + 16.0f * q[j + 1];
                if (UV<T> > 2) four += 256.0f * (q[(j + 2) % UV<T>] + 16.0f * q[(j + 3) % UV<T>]);
                code[0] |= (uint32_t)four << (4 * j);
            }
            put_code<UV<T> / 2, (S > 1)>(row + u * (UV<T> / 2), code);
        }
    }
    if (y) {
#pragma unroll
        for (int j = 0; j < UV<T>; j++) out.v[j] = narrow<T>(dequantise(q[j], s, W(0)));
        out.template store<(S > 0)>(y + (int64_t)u * UV<T>, n);
    }
}

// A frame -- or, of a wide grouped one, a segment of it -- lies in the registers of its lanes (Spread).  Its extremes are joined across
// those lanes (a group's across the lanes of the group), the codes follow from the same registers: the frames are read once.  Bound by
// HBM in fp32 and fp64: 102 400 x 192 bands of fp32 to 8 bits with values 56 us (6.3 TB/s) into slots in order, 60 with the claims
// of slots in any order; 409 600 of fp64 to 4 bits 440 us (5.95 TB/s).  16-bit types are bound by the vector unit as
// well: 409 600 of bf16 to 8 bits 109 us without values (77 for the bytes; 421 instructions a wave, 70 us of issue) and 159 with (128; 489),
// in groups of 64 bands 119 (602, 100 us: each unit's lanes work their group's scale out) and 159 (669), of 16 bands 126 and 171.
template <class T, int NC, bool GROUPED, int S> __global__ __launch_bounds__(256) void k_write(WriteArgs a) {
    typedef typename Wide<T>::type W;
    const int lanes = 1 << a.p.lanes_log2, l = (int)threadIdx.x & (lanes - 1);
    const int64_t part = (a.block0 + blockIdx.x) * (256 >> a.p.lanes_log2) + ((int)threadIdx.x >> a.p.lanes_log2);
    if (part >= a.n * a.p.segs) return;
    const int64_t r = a.p.segs == 1 ? part : part / a.p.segs;
    const int u0 = a.p.segs == 1 ? 0 : (int)(part - r * a.p.segs) * (NC * lanes);
    const int64_t slot = slot_of(a.slots, r);   // before the frame's loads: the claim hangs on it and comes while they are on their way
    const T* x = (const T*)a.x + r * a.xs;
    Unit<T> in[NC];
    int n[NC];
#pragma unroll
    for (int k = 0; k < NC; k++) {
        const int c = (u0 + l + k * lanes) * UV<T>;
        n[k] = min(UV<T>, 2 * a.l.K - c);
        if (n[k] > 0) in[k] = Unit<T>::template load<(S > 0)>(x + c, n[k]);
    }
    if (slot < 0 || slot >= a.slots.n_slots) {
        if (slot >= a.slots.n_slots && l == 0 && u0 == 0) atomicAdd(a.bad, 1ull);
        return;
    }
    const int first = (int)(threadIdx.x & 63) & ~(lanes - 1);   // of this frame's lanes in the wave
    int32_t owner = (int32_t)r;
    if (a.claim) owner = claim_of(a.claim + slot);
    else if (a.slots.at && a.n > 1) {
        bool again = false;
        for (int i = (int)r + 1 + l; i < (int)a.n; i += 8 * lanes) {   // eight loads in flight: one at a time costs 0.1 us each
            int64_t at[8];
#pragma unroll
            for (int k = 0; k < 8; k++) at[k] = a.slots.at[min(i + k * lanes, (int)a.n - 1)];
#pragma unroll
            for (int k = 0; k < 8; k++) again |= at[k] == slot && i + k * lanes < (int)a.n;
        }
        if (__ballot(again) >> first & (~0ull >> (64 - lanes))) owner = -1;
    }
    uint8_t* row = a.store + slot * a.l.row_bytes;
    T* y = a.y ? (T*)a.y + r * a.ys : nullptr;
    W w[NC][UV<T>];
    Range<W> range[GROUPED ? NC : 1];
#pragma unroll
    for (int k = 0; k < NC; k++) {
        if (n[k] <= 0) continue;
#pragma unroll
        for (int j = 0; j < UV<T>; j++) w[k][j] = widen(in[k].v[j]);
#pragma unroll
        for (int j = 0; j < UV<T>; j += 2) range[GROUPED ? k : 0].add(w[k][j], w[k][j + 1]);
    }
    const bool keep = owner == (int32_t)r;
    const int span = GROUPED ? 1 << a.gunits_log2 : lanes;          // lanes that hold a group
    const int start = (int)(threadIdx.x & 63) & ~(span - 1);
    const int levels = (1 << a.l.bits) - 1;
#pragma unroll
    for (int g = 0; g < (GROUPED ? NC : 1); g++) {
        W mn = range[g].mn, mx = range[g].mx;
        join(span, &mn, &mx);
        int flags = 0;
        if (__ballot(range[g].special()) >> start & (~0ull >> (64 - span))) {
            mn = (W)__builtin_inf(); mx = -(W)__builtin_inf();
#pragma unroll
            for (int k = GROUPED ? g : 0; k < (GROUPED ? g + 1 : NC); k++)
#pragma unroll
                for (int j = 0; j < UV<T>; j++) if (n[k] > 0) add_finite(w[k][j], &mn, &mx, &flags);
            join(span, &mn, &mx);
            for (int m = 1; m < span; m <<= 1) flags |= __shfl_xor(flags, m);
        }
        const Scale s = group_scale(mn, mx, flags, levels);
        const W per = reciprocal(s, W(0));
        const int ug = u0 + l + g * lanes;                          // GROUPED: the unit whose group this is
        if (keep && (GROUPED ? ((ug & (span - 1)) == 0 && n[g] > 0) : l == 0))
            *(float2*)(row + a.l.scale_off + 8 * (GROUPED ? ug >> a.gunits_log2 : 0)) = make_float2(s.lo, s.step);
#pragma unroll
        for (int k = GROUPED ? g : 0; k < (GROUPED ? g + 1 : NC); k++)
            if (n[k] > 0) put_unit<T, S>(a, row, y, keep, u0 + l + k * lanes, n[k], w[k], s, per);
    }
    if (a.claim && keep && l == 0 && a.p.segs == 1) a.claim[slot] = -1;   // (a frame that lost reads its rival's index or this: neither is its own)
}

// A frame under one scale that is too wide for a wave's registers: a block per frame, which reads it twice (the second time out of the
// caches: at most 256 KB).  4 000 x 2 600 bands of fp32 to 8 bits 32 us (17 for the bytes), 40 000 with values 415 (302).
template <class T> __global__ __launch_bounds__(256) void k_write_wide(WriteArgs a) {
    typedef typename Wide<T>::type W;
    __shared__ W s_mn[4], s_mx[4];
    __shared__ int s_flags[4];
    const int64_t r = a.block0 + blockIdx.x, slot = slot_of(a.slots, r);
    const int t = (int)threadIdx.x, cols = 2 * a.l.K;
    if (slot < 0 || slot >= a.slots.n_slots) {
        if (slot >= a.slots.n_slots && t == 0) atomicAdd(a.bad, 1ull);
        return;
    }
    bool keep = true;
    if (a.claim) {
        keep = claim_of(a.claim + slot) == (int32_t)r;
        __syncthreads();
        if (keep && t == 0) a.claim[slot] = -1;
    } else if (a.slots.at && a.n > 1) {
        int again = 0;
        for (int64_t i = r + 1 + t; i < a.n; i += 256) again |= a.slots.at[i] == slot;
        keep = !__syncthreads_or(again);
    }
    const T* x = (const T*)a.x + r * a.xs;
    W mn = (W)__builtin_inf(), mx = -(W)__builtin_inf();
    int flags = 0;
    for (int c = t * UV<T>; c < cols; c += 256 * UV<T>) {
        const int n = min(UV<T>, cols - c);
        const Unit<T> in = Unit<T>::template load<false>(x + c, n);
#pragma unroll
        for (int j = 0; j < UV<T>; j++) add_finite(widen(in.v[j]), &mn, &mx, &flags);
    }
    join(64, &mn, &mx);
    for (int m = 1; m < 64; m <<= 1) flags |= __shfl_xor(flags, m);
    if ((t & 63) == 0) { s_mn[t >> 6] = mn; s_mx[t >> 6] = mx; s_flags[t >> 6] = flags; }
    __syncthreads();
    for (int i = 0; i < 4; i++) { mn = least(mn, s_mn[i]); mx = most(mx, s_mx[i]); flags |= s_flags[i]; }
    const Scale s = group_scale(mn, mx, flags, (1 << a.l.bits) - 1);
    const W per = reciprocal(s, W(0));
    uint8_t* row = a.store + slot * a.l.row_bytes;
    T* y = a.y ? (T*)a.y + r * a.ys : nullptr;
    if (keep && t == 0) *(float2*)(row + a.l.scale_off) = make_float2(s.lo, s.step);
    for (int c = t * UV<T>; c < cols; c += 256 * UV<T>) {
        const int n = min(UV<T>, cols - c);
        const Unit<T> in = Unit<T>::template load<false>(x + c, n);
        W w[UV<T>];
#pragma unroll
        for (int j = 0; j < UV<T>; j++) w[j] = widen(in.v[j]);
        put_unit<T, 0>(a, row, y, keep, c / UV<T>, n, w, s, per);
    }
}

// The 32 random bits of the N elements from `e` on: one word of the generator for two elements, its argument stepped from word to word;
// an odd start straddles words and needs one more.  The word's index has 63 bits: where the element's 64 wrap to zero (`wraps`: the call
// reaches there) the stepped argument is 2^63 kGamma = 2^63 too large.
template <int N> GL_DEV void random_bits(uint64_t seed, uint64_t e, bool wraps, uint32_t* u) {
    const uint64_t i = e >> 1;
    const bool odd = e & 1;
    uint64_t z[N / 2 + 1], w[N / 2 + 1];
    z[0] = seed + (i + 1) * kGamma;
#pragma unroll
    for (int j = 1; j <= N / 2; j++) z[j] = z[j - 1] + kGamma;
    if (wraps) {
#pragma unroll
        for (int j = 1; j <= N / 2; j++) z[j] ^= (i + j) & ((uint64_t)1 << 63);
    }
#pragma unroll
    for (int j = 0; j < N / 2; j++) w[j] = splitmix_of(z[j]);
    w[N / 2] = 0;
    if (odd) w[N / 2] = splitmix_of(z[N / 2]);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        u[j] = odd ? (uint32_t)(w[j / 2] >> 32) : (uint32_t)w[j / 2];
        u[j + 1] = odd ? (uint32_t)w[j / 2 + 1] : (uint32_t)(w[j / 2] >> 32);
    }
}
template <class T> GL_DEV T drop_or(typename Wide<T>::type v, const DropRule& d, uint32_t u) {
    typedef typename Wide<T>::type W;
    const bool all = d.all != 0, low = u < d.below;
    return narrow<T>((all | low) ? W(0) : v * (W)d.scale);
}

// What k_read and k_read_drop share: the frame this lane works on, its first unit there, the frame's row in the cache; false: none.
GL_DEV bool read_place(const ReadArgs& a, int units, int64_t* r, int* u0, const uint8_t** row) {
    const int lanes = 1 << a.p.lanes_log2, l = (int)threadIdx.x & (lanes - 1);
    const int64_t part = (a.block0 + blockIdx.x) * (256 >> a.p.lanes_log2) + ((int)threadIdx.x >> a.p.lanes_log2);
    if (part >= a.n * a.p.segs) return false;
    *r = a.p.segs == 1 ? part : part / a.p.segs;
    *u0 = (a.p.segs == 1 ? 0 : (int)(part - *r * a.p.segs) * (units * lanes)) + l;
    const int64_t slot = slot_of(a.slots, *r);
    if (slot < 0 || slot >= a.slots.n_slots) {
        if ((slot >= a.slots.n_slots || a.strict) && *u0 == 0) atomicAdd(a.bad, 1ull);
        return false;
    }
    *row = a.store + slot * a.l.row_bytes;
    return true;
}
// A unit's codes: a row's are padded to 16 bytes, so a partial unit's are there too.
template <class T, int BITS> struct Codes {
    static constexpr int bytes = UV<T> * BITS / 8;
    uint32_t v[bytes > 4 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* row, int u) {
        v[0] = 0;
        __builtin_memcpy(v, __builtin_assume_aligned(row + u * bytes, bytes), bytes);
    }
    __device__ __forceinline__ float at(int j) const { return (float)(v[j * BITS / 32] >> (j * BITS % 32) & ((1u << BITS) - 1)); }
};

// A frame over the lanes as in k_write.  Per unit: its codes (1 ... 8 bytes), its group's scale, one 16-byte store.  Bound by HBM: 102 400 x
// 192 bands from 4 bits to fp32 28 us (6.7 TB/s), 409 600 from 8 bits to bf16 82 us (5.9 TB/s) in order, 89 in pages of 16 in any order.
template <class T, int BITS, int NC, bool S> __global__ __launch_bounds__(256) void k_read(ReadArgs a) {
    typedef typename Wide<T>::type W;
    int64_t r;
    int u0;
    const uint8_t* row;
    if (!read_place(a, NC, &r, &u0, &row)) return;
    const int lanes = 1 << a.p.lanes_log2;
    const float2* scales = (const float2*)(row + a.l.scale_off);
    Codes<T, BITS> code[NC];
    float2 f[NC];
    int n[NC];
#pragma unroll
    for (int k = 0; k < NC; k++) {
        const int u = u0 + k * lanes;
        n[k] = min(UV<T>, 2 * a.l.K - u * UV<T>);
        if (n[k] <= 0) continue;
        code[k].load(row, u);
        f[k] = scales[(u * UV<T> >> 1) >> a.gshift];
    }
    T* y = (T*)a.y + r * a.ys;
#pragma unroll
    for (int k = 0; k < NC; k++) {
        if (n[k] <= 0) continue;
        Unit<T> out;
#pragma unroll
        for (int j = 0; j < UV<T>; j++) out.v[j] = narrow<T>(dequantise(code[k].at(j), Scale{f[k].x, f[k].y}, W(0)));
        out.template store<S>(y + (u0 + k * lanes) * UV<T>, n[k]);
    }
}
// The same with dropout: bound by the generator as dropout in 16 bits is (54 912 x 80 bands to bf16: 8.8 us, of which 5.6 are its products),
// so the lane's units go through one loop body; loading the next unit's codes ahead changed nothing.  102 400 x 192 bands: bf16 23.5 us,
// fp32 30.4 (6.5 TB/s) and fp64 49.4 (7.2, codes partly from the caches): there HBM is the bound.
template <class T, int BITS, bool S> __global__ __launch_bounds__(256) void k_read_drop(ReadArgs a) {
    typedef typename Wide<T>::type W;
    int64_t r;
    int u0;
    const uint8_t* row;
    if (!read_place(a, a.p.units, &r, &u0, &row)) return;
    const float2* scales = (const float2*)(row + a.l.scale_off);
    T* y = (T*)a.y + r * a.ys;
    const uint64_t e = a.offset + (uint64_t)r * (uint32_t)(2 * a.l.K);
#pragma unroll 1
    for (int k = 0; k < a.p.units; k++) {
        const int c = (u0 + (k << a.p.lanes_log2)) * UV<T>, n = min(UV<T>, 2 * a.l.K - c);
        if (n <= 0) return;
        Codes<T, BITS> code;
        code.load(row, c / UV<T>);
        const float2 f = scales[(c >> 1) >> a.gshift];
        uint32_t bits[UV<T>];
        random_bits<UV<T>>(a.seed, e + (uint32_t)c, a.wraps, bits);
        Unit<T> out;
#pragma unroll
        for (int j = 0; j < UV<T>; j++) {
            out.v[j] = drop_or<T>(dequantise(code.at(j), Scale{f.x, f.y}, W(0)), a.drop, bits[j]);
        }
        out.template store<S>(y + c, n);
    }
}

struct DropArgs {
    const void* x; void* y;
    int64_t xs, ys, cols, total;
    Walk w;
    DropRule drop;
    uint64_t seed, offset;
    int32_t wraps;            // offset + total pass 2^64
    int64_t block0 = 0;
};
// Dense arrays: one unit per lane.  Bound by HBM in fp32 and fp64 (two streams), by the generator's multiplications in the 16-bit types:
// six quarter-rate 32-bit products for two elements.  One unit per lane is the best of 1, 2, 4 and 8: with more in flight per lane
// fp32 falls from 6.17 to 5.9 TB/s, bf16 from 6.08 to 5.8 (409 600 x 384 elements, bytes read and written).
template <class T, bool S, bool LN> __global__ __launch_bounds__(256) void k_dropout(DropArgs a) {
    const int64_t e0 = (a.block0 + blockIdx.x) * (256 * UV<T>);
    const int t = (int)threadIdx.x * UV<T>;
    const int n = (int)min((int64_t)UV<T>, a.total - e0 - t);
    if (n <= 0) return;
    Unit<T> x = Unit<T>::template load<LN>((const T*)a.x + e0 + t, n);
    uint32_t u[UV<T>];
    random_bits<UV<T>>(a.seed, a.offset + (uint64_t)e0 + (uint32_t)t, a.wraps, u);
#pragma unroll
    for (int j = 0; j < UV<T>; j++) x.v[j] = drop_or<T>(widen(x.v[j]), a.drop, u[j]);
    x.template store<S>((T*)a.y + e0 + t, n);
}
// Rows apart, each with units of its own (Walk).  102 400 rows of 384 elements 390 apart: bf16 25.9 us, fp32 55.2 (6.1 and 5.7 TB/s); of 322,
// 384 apart: 34.8 and 49.7 (3.8 and 5.3): a 41st unit of two elements to every row.
template <class T, bool S> __global__ __launch_bounds__(512) void k_dropout_rows(DropArgs a) {
    int64_t r, k;
    if (!walk_unit(a.w, a.block0 + blockIdx.x, &r, &k)) return;
    const int64_t c = k * UV<T>;
    const int n = (int)min((int64_t)UV<T>, a.cols - c);
    Unit<T> x = Unit<T>::template load<false>((const T*)a.x + r * a.xs + c, n);
    const uint64_t e = a.offset + (uint64_t)(r * a.cols + c);
    uint32_t u[UV<T>];
    random_bits<UV<T>>(a.seed, e, a.wraps, u);
#pragma unroll
    for (int j = 0; j < UV<T>; j++) x.v[j] = drop_or<T>(widen(x.v[j]), a.drop, u[j]);
    x.template store<S>((T*)a.y + r * a.ys + c, n);
}

#define GL_TYPES(type, ...)                                          \
    switch (type) {                                                  \
        case GOMEL_F64: { typedef double T; __VA_ARGS__; } break;    \
        case GOMEL_F32: { typedef float T; __VA_ARGS__; } break;     \
        case GOMEL_F16: { typedef __half T; __VA_ARGS__; } break;    \
        default: { typedef __hip_bfloat16 T; __VA_ARGS__; } break;   \
    }
template <class T, bool G, int S> void (*write_kernel(int units))(WriteArgs) {
    switch (units) {
        case 1: return k_write<T, 1, G, S>;
        case 2: return k_write<T, 2, G, S>;
        case 3: return k_write<T, 3, G, S>;
        case 4: return k_write<T, 4, G, S>;
        case 5: return k_write<T, 5, G, S>;
        default: return k_write<T, 6, G, S>;
    }
}
template <class T> void (*write_kernel(int units, bool grouped, int streamed))(WriteArgs) {
    if (grouped) return streamed == 2 ? write_kernel<T, true, 2>(units) : streamed ? write_kernel<T, true, 1>(units) : write_kernel<T, true, 0>(units);
    return streamed == 2 ? write_kernel<T, false, 2>(units) : streamed ? write_kernel<T, false, 1>(units) : write_kernel<T, false, 0>(units);
}
template <class T, int BITS, bool S> void (*read_kernel(int units, bool dropping))(ReadArgs) {
    if (dropping) return k_read_drop<T, BITS, S>;
    switch (units) {
        case 1: return k_read<T, BITS, 1, S>;
        case 2: return k_read<T, BITS, 2, S>;
        case 3: return k_read<T, BITS, 3, S>;
        case 4: return k_read<T, BITS, 4, S>;
        case 5: return k_read<T, BITS, 5, S>;
        default: return k_read<T, BITS, 6, S>;
    }
}
template <class T> void (*read_kernel(int bits, int units, bool dropping, bool streamed))(ReadArgs) {
    if (bits == 8) return streamed ? read_kernel<T, 8, true>(units, dropping) : read_kernel<T, 8, false>(units, dropping);
    return streamed ? read_kernel<T, 4, true>(units, dropping) : read_kernel<T, 4, false>(units, dropping);
}
// Large outputs are stored past the caches (non-temporal): left in them, their write-back is in the way of the kernels that follow.  A
// read of 102 400 x 192 bands (157 MB of fp32) takes 28.4 us instead of 45.3, 50.7 instead of 94.7 in fp64, a write with its values 62
// instead of 80, dropout of 79 MB of bf16 23.8 instead of 29.0, each among others of its kind; with a consumer right behind that could
// have found the output in the 256 MB last-level cache, the pair gains (write, dropout: up to 9 %) or loses (read: up to 5 %).  Below a
// quarter of that cache nothing is gained.  Frames to be written are loaded so too, dropout's input where input and output together do
// not fit (315 MB of fp32: 194.9 instead of 199.2 us; 79 MB: 26.7 instead of 23.8).
constexpr size_t kStreamBytes = (size_t)64 << 20, kStreamInBytes = (size_t)128 << 20;
// A launch has fewer than 2^32 lanes: grids of more blocks go out in parts, a block's index counted on through them (`block0`).  Launches
// report their own status: hipGetLastError could hand back somebody else's.
constexpr size_t kBlocks = (size_t)1 << 22;
thread_local int g_fail_launch = 0;   // gomel_debug_fail_launch
template <class Args> hipError_t launch(void (*k)(Args), size_t blocks, unsigned block, hipStream_t s, Args& a) {
    hipError_t e = hipSuccess;
    for (size_t b = 0; b < blocks && e == hipSuccess; b += kBlocks) {
        if (g_fail_launch && --g_fail_launch == 0) return hipErrorLaunchFailure;
        a.block0 = (int64_t)b;
        void* p[] = {&a};
        e = hipLaunchKernel((const void*)k, dim3((unsigned)std::min(kBlocks, blocks - b)), dim3(block), p, 0, s);
    }
    return e;
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
int hip_failed(hipError_t e) { set_last_hip((int)e); (void)hipGetLastError(); return GOMEL_ERR_HIP; }
#define CHK(expr) do { const hipError_t e_ = (expr); if (e_ != hipSuccess) return hip_failed(e_); } while (0)

hipError_t dropout_device(int type, const void* x, size_t xs, void* y, size_t ys, size_t rows, size_t cols, const DropRule& d, uint64_t seed, uint64_t offset, hipStream_t s) {
    const size_t total = rows * cols, bytes = total * (size_t)type_bytes(type), uv = 16 / (size_t)type_bytes(type);
    DropArgs a{x, y, (int64_t)xs, (int64_t)ys, (int64_t)cols, (int64_t)total, Walk{}, d, seed, offset, (int32_t)(offset + (uint64_t)total < offset)};
    hipError_t e = hipSuccess;
    if ((xs == cols && ys == cols) || rows == 1) {
        const size_t units = (total + uv - 1) / uv, blocks = (units + 256 - 1) / 256;
        GL_TYPES(type, e = launch(bytes < kStreamBytes ? k_dropout<T, false, false> : bytes < kStreamInBytes ? k_dropout<T, true, false> : k_dropout<T, true, true>,
                                  blocks, 256, s, a));
        return e;
    }
    a.w = walk_of(rows, (cols + uv - 1) / uv);
    GL_TYPES(type, e = launch(bytes < kStreamBytes ? k_dropout_rows<T, false> : k_dropout_rows<T, true>, (size_t)a.w.blocks, (unsigned)a.w.block, s, a));
    return e;
}

constexpr size_t kStageBytes = (size_t)32 << 20;
// Frames of a write up to which each looks through the later slots itself, per lane that looks; more claim theirs first.  The search grows
// with the square, the claims cost a launch (192 bands of bf16, slots in any order: 64 lanes look, 6.0 us for 1 024 and for 2 048 frames, 8.9
// for 4 096; by claims 8 192 frames 9.1; in slot order, with neither, 5.6 ... 6.5.  16 lanes took 10.2 for 2 048).
constexpr size_t kScanPerLane = 64;

// Rows between host memory (stride elements apart) and a dense device buffer
hipError_t rows_in(void* dev, const char* host, size_t stride, size_t rows, size_t cols, size_t esz, hipStream_t s) {
    if (stride == cols || rows == 1) return hipMemcpyAsync(dev, host, rows * cols * esz, hipMemcpyDefault, s);
    return hipMemcpy2DAsync(dev, cols * esz, host, stride * esz, cols * esz, rows, hipMemcpyDefault, s);
}
hipError_t rows_out(char* host, const void* dev, size_t stride, size_t rows, size_t cols, size_t esz, hipStream_t s) {
    if (stride == cols || rows == 1) return hipMemcpyAsync(host, dev, rows * cols * esz, hipMemcpyDefault, s);
    return hipMemcpy2DAsync(host, stride * esz, dev, cols * esz, cols * esz, rows, hipMemcpyDefault, s);
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
    const bool vouched = type & GOMEL_DEVICE_MEMORY;
    type &= ~GOMEL_DEVICE_MEMORY;
    const size_t cols = 2 * (size_t)c->l.K, esz = (size_t)type_bytes(type);
    if (!esz) return GOMEL_ERR_BAD_CONFIG;
    if (n == 0) return GOMEL_OK;
    if (n > kMaxRows || (in && !rows_span(n, cols, is)) || (out && !rows_span(n, cols, os))) return GOMEL_ERR_BAD_LENGTH;
    if (!slots && (first > c->n_slots || n > c->n_slots - first)) return GOMEL_ERR_TABLE_RANGE;
    if ((uintptr_t)in % esz || (uintptr_t)out % esz || (uintptr_t)slots % 8) return GOMEL_ERR_BAD_CONFIG;
    if (in && out && !rows_disjoint_or_same(in, is, out, os, n, cols, esz)) return GOMEL_ERR_BAD_CONFIG;
    OnDevice dev(c->device); CHK(dev.err);
    if (vouched) { CHK(run(type, in, is, out, os, n, slots, first)); return GOMEL_OK; }
    const int ki = in ? memory_kind(in, c->device) : 1, ko = out ? memory_kind(out, c->device) : 1, ks = slots ? memory_kind(slots, c->device) : 1;
    if (ki < 0 || ko < 0 || ks < 0) return GOMEL_ERR_BAD_CONFIG;
    if (ki && ko && ks) { CHK(run(type, in, is, out, os, n, slots, first)); return GOMEL_OK; }
    if (stream_capturing(s)) return GOMEL_ERR_BAD_CONFIG;
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
        if (!ks) e = hipMemcpyAsync(st_slots, at, m * 8, hipMemcpyDefault, s);
        if (!ki && e == hipSuccess) e = rows_in(st, from, is, m, cols, esz, s);
        if (!ko && slots && e == hipSuccess) e = rows_in(st_out, to, os, m, cols, esz, s);   // rows of padding come back as they were
        if (e == hipSuccess) e = run(type, ki ? from : st, ki ? is : cols, ko ? to : st_out, ko ? os : cols, m, ks ? at : (const int64_t*)st_slots, first + r);
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
    // one allocation: rows | claims | count of bad slots
    const size_t rows = (n_slots * (size_t)l.row_bytes + 255) & ~(size_t)255, claims = (n_slots * 4 + 255) & ~(size_t)255;
    if (e == hipSuccess) e = hipMalloc((void**)&c->store, rows + claims + 256);
    if (e == hipSuccess) {
        const hipStream_t s = handle_stream(h);   // not the default stream, which would wait for everybody's work
        c->claim = (int32_t*)(c->store + rows);
        c->bad = (unsigned long long*)(c->store + rows + claims);
        e = hipMemsetAsync(c->store, 0, rows, s);
        if (e == hipSuccess) e = hipMemsetAsync(c->claim, 0xFF, claims, s);
        if (e == hipSuccess) e = hipMemsetAsync(c->bad, 0, 8, s);
        const hipError_t e2 = hipStreamSynchronize(s);
        if (e == hipSuccess) e = e2;
    }
    if (e != hipSuccess) {
        if (c->store) (void)hipFree(c->store);
        delete c;
        return hip_failed(e);
    }
    *out = c;
    return GOMEL_OK;
}

int dropout_call(gomel_handle* h, int type, const void* x, size_t xs, void* y, size_t ys, size_t rows, size_t cols, double p, uint64_t seed, uint64_t offset, hipStream_t s) {
    if (!h) return GOMEL_ERR_NULL;
    const bool vouched = type & GOMEL_DEVICE_MEMORY;
    type &= ~GOMEL_DEVICE_MEMORY;
    const size_t esz = (size_t)type_bytes(type);
    DropRule d;
    if (!esz || !drop_rule(p, &d)) return GOMEL_ERR_BAD_CONFIG;
    if (rows == 0 || cols == 0) return GOMEL_OK;
    if (!x || !y) return GOMEL_ERR_NULL;
    if (!rows_span(rows, cols, xs) || !rows_span(rows, cols, ys)) return GOMEL_ERR_BAD_LENGTH;
    if ((uintptr_t)x % esz || (uintptr_t)y % esz || !rows_disjoint_or_same(x, xs, y, ys, rows, cols, esz)) return GOMEL_ERR_BAD_CONFIG;
    const int device = handle_device(h);
    OnDevice dev(device); CHK(dev.err);
    const int kx = vouched ? 1 : memory_kind(x, device), ky = vouched ? 1 : memory_kind(y, device);
    if (kx < 0 || ky < 0) return GOMEL_ERR_BAD_CONFIG;
    if (kx && ky) { CHK(dropout_device(type, x, xs, y, ys, rows, cols, d, seed, offset, s)); return GOMEL_OK; }
    if (stream_capturing(s)) return GOMEL_ERR_BAD_CONFIG;
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

bool stream_capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (!s) return false;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) { (void)hipGetLastError(); return false; }
    return st != hipStreamCaptureStatusNone;
}

hipError_t cache_write_device(gomel_cache* c, int type, const void* x, size_t xs, size_t n, const int64_t* slots, size_t first, void* y, size_t ys, hipStream_t s) {
    const bool grouped = c->l.groups > 1;
    const int uv = 16 / type_bytes(type), upr = (2 * c->l.K + uv - 1) / uv;
    int gunits_log2 = 0;
    if (grouped) while ((uv << gunits_log2) < 2 * c->l.group) gunits_log2++;
    const Spread p = spread_of(n, upr, std::max(3, gunits_log2), grouped);
    const bool claims = slots && n > (p.units ? kScanPerLane << p.lanes_log2 : 2048);
    WriteArgs a{x, y, (int64_t)xs, (int64_t)ys, (int64_t)n, Slots{slots, (int64_t)first, (int64_t)c->n_slots}, c->store, c->l, claims ? c->claim : nullptr, c->bad, p, gunits_log2};
    hipError_t e = hipSuccess;
    if (claims) e = launch_claim(k_claim, a.slots, a.n, c->claim, s);
    if (e != hipSuccess) return e;
    if (!a.p.units) {
        GL_TYPES(type, e = launch(k_write_wide<T>, n, 256, s, a));
    } else {
        const size_t per = 256 >> a.p.lanes_log2, blocks = (n * (size_t)a.p.segs + per - 1) / per;
        const int streamed = 2 * (size_t)c->l.K * n * type_bytes(type) < kStreamBytes ? 0 : n * (size_t)c->l.row_bytes < kStreamInBytes ? 1 : 2;
        GL_TYPES(type, e = launch(write_kernel<T>(a.p.units, grouped, streamed), blocks, 256, s, a));
    }
    // a write that was not launched, or not all of it, leaves claims standing: a later call's lower rows would lose to them
    if (claims && (a.p.segs > 1 || e != hipSuccess)) {
        const hipError_t e2 = launch_claim(k_claim_clear, a.slots, a.n, c->claim, s);
        if (e == hipSuccess) e = e2;
    }
    return e;
}

hipError_t cache_read_device(gomel_cache* c, int type, void* y, size_t ys, size_t n, const int64_t* slots, size_t first, const DropRule& drop,
                             uint64_t seed, uint64_t offset, bool strict, unsigned long long* bad, hipStream_t s) {
    const int uv = 16 / type_bytes(type);
    int gshift = 31;
    if (c->l.groups > 1) for (gshift = 0; (1 << gshift) < c->l.group; gshift++) {}
    ReadArgs a{y, (int64_t)ys, (int64_t)n, Slots{slots, (int64_t)first, (int64_t)c->n_slots}, c->store, c->l, spread_of(n, (2 * c->l.K + uv - 1) / uv, 3, true), drop,
               gshift, (int32_t)strict, seed, offset, bad ? bad : c->bad, (int32_t)(offset + 2 * (uint64_t)c->l.K * n < offset)};
    const size_t per = 256 >> a.p.lanes_log2, blocks = (n * (size_t)a.p.segs + per - 1) / per;
    const bool dropping = drop.all || drop.below != 0 || drop.scale != 1.0;   // (p below 2^-33 drops nothing, its factor stays)
    hipError_t e = hipSuccess;
    GL_TYPES(type, e = launch(read_kernel<T>(c->l.bits, a.p.units, dropping, 2 * (size_t)c->l.K * n * type_bytes(type) >= kStreamBytes), blocks, 256, s, a));
    return e;
}

// ------------------------------------------------------------------------------------------------ C ABI
extern "C" {

// Diagnostics (not in the header; the tests reach it by name): what every call here returns when the runtime failed with `e`.
int gomel_debug_hip_failed(int e) { return hip_failed((hipError_t)e); }
// Diagnostics (not in the header; the tests reach it by name): the calling thread's n-th launch of a write, read or dropout kernel from now
// on fails without being launched, as one that the runtime refuses would.  0: none.
void gomel_debug_fail_launch(int n) { g_fail_launch = n; }

int gomel_cache_create(gomel_handle* h, size_t n_slots, int bits, int group_bands, gomel_cache** out) {
    GOMEL_TRY return cache_create(h, n_slots, bits, group_bands, out); GOMEL_CATCH
}

int gomel_cache_destroy(gomel_cache* c) {
    if (!c) return GOMEL_OK;
    {
        OnDevice dev(c->device);
        hipError_t e = hipDeviceSynchronize();   // calls only queue work: it may still be running on any stream
        for (void* p : {(void*)c->store, c->stage}) {
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
                      [&](int t, const void* in, size_t is, void* out, size_t os, size_t m, const int64_t* at, size_t f) { return cache_write_device(c, t, in, is, m, at, f, out, os, s); });
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
    return cache_call(c, type, nullptr, 0, frames, stride, n, slots, first, s, [&](int t, const void*, size_t, void* out, size_t os, size_t m, const int64_t* at, size_t f) {
        const hipError_t e = cache_read_device(c, t, out, os, m, at, f, d, seed, offset + done * cols, false, nullptr, s);
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
    hipError_t e = hipMemcpyAsync(&got, c->bad, 8, hipMemcpyDeviceToHost, s);   // never set back: a running call may be counting
    const hipError_t e2 = hipStreamSynchronize(s);
    (void)hipStreamDestroy(s);
    if (e == hipSuccess) e = e2;
    if (e != hipSuccess) return hip_failed(e);
    *count = got - c->told;
    c->told = got;
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
