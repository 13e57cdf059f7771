// What the trainable frame operators (selective scan, short convolution, layer norm, gradient
// clipping) share: element types of two and four bytes, vector loads and stores that need no more
// than the element's own alignment, sums over parts of a wave, and the guard that leaves the
// caller's current device as it was.
#pragma once
#include "srx_internal.h"

#include <string.h>

namespace srx_frames {

template <typename T, int V>
struct Pack {
    typedef T Vec __attribute__((ext_vector_type(V)));
    Vec v;
};

// V neighbouring elements as one memory instruction: gfx950 takes global accesses at any
// alignment, and full width where the address happens to be aligned.
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    Pack<T, V> r;
    __builtin_memcpy(&r.v, (const void*)p, V * sizeof(T));
    return r;
}
template <int V, typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    __builtin_memcpy((void*)p, &v.v, V * sizeof(T));
}
// The same at a scalar global address plus a 32-bit offset of the lane's own: one scalar register pair and one
// vector register, instead of a 64-bit address in vector registers.  (The scalar part is hidden from the optimiser, which
// would add the two up.)
typedef __attribute__((address_space(1))) char GlobalChar;
__device__ __forceinline__ GlobalChar* global_at(GlobalChar* base, unsigned off) {
    asm("" : "+s"(base));
    asm("" : "+v"(off));
    return base + off;
}
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_global(GlobalChar* base, unsigned off) {
    typedef typename Pack<T, V>::Vec Vec;
    typedef Vec Loose __attribute__((aligned(sizeof(T))));
    Pack<T, V> r;
    r.v = *(__attribute__((address_space(1))) const Loose*)global_at(base, off);
    return r;
}
template <int V, typename T>
__device__ __forceinline__ void store_global(GlobalChar* base, unsigned off, const Pack<T, V>& v) {
    typedef typename Pack<T, V>::Vec Vec;
    typedef Vec Loose __attribute__((aligned(sizeof(T))));
    *(__attribute__((address_space(1))) Loose*)global_at(base, off) = v.v;
}
// The first `n` (<= V) of V neighbouring elements, zeros behind them.
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_some(const T* p, int n) {
    if (n >= V) return load_pack<V>(p);
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : (T)0.0f;
    return r;
}
template <int V, typename T>
__device__ __forceinline__ void store_some(T* p, const Pack<T, V>& v, int n) {
    if (n >= V) {
        store_pack(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) p[i] = v.v[i];
}

// The same where a condition that holds for the whole wave says that all V exist: a branch that the wave takes as one, so
// that a row of such loads stays one run of instructions and all of them are in flight together.
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_where(bool all, const T* p, int n) {
    if (all) return load_pack<V>(p);
    return load_some<V>(p, n);
}
template <int V, typename T>
__device__ __forceinline__ void store_where(bool all, T* p, const Pack<T, V>& v, int n) {
    if (all) store_pack(p, v);
    else store_some(p, v, n);
}

// e^x by the hardware's 2^x; the part of x log2(e) that its rounding to 32 bits drops is put
// back to first order, so that the relative error does not grow with |x|.  0 and infinity stay as they are: they have no
// such error, and where the product itself overflows there is no dropped part (it would come out as NaN).
__device__ __forceinline__ float exp_f32(float x) {
    const float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147180559945309f;
    const float t = x * kLog2e;
    const float rest = fmaf(x, kLog2e, -t) + x * kLog2eRest;
    const float e = __builtin_amdgcn_exp2f(t);
    return e > 0.0f && e < __builtin_huge_valf() ? fmaf(e, rest * kLn2, e) : e;
}
__device__ __forceinline__ float sigmoid_f32(float x) {
    // (the exponential overflows to infinity for x below -88, the quotient is then zero)
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x));
}
// ln(1 + e^x) = max(x, 0) + log1p(e^-|x|).  log1p(e): the logarithm of u = 1 + e, plus what the rounding
// of that sum dropped, which for a small e is most of its relative accuracy (steps of 0.001 and less
// are ordinary); its derivative 1 / u is taken as 1, as the dropped part is below 2^-24.  The exponential is
// off by |x| 2^-24 of itself, as much as x is when it is itself a rounded sum.  A NaN comes through the exponential.
// slope: its derivative, the sigmoid, from the same exponential.
__device__ __forceinline__ float softplus_f32(float x, float& slope) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * fabsf(x));
    const float u = 1.0f + e;
    const float inverse = __builtin_amdgcn_rcpf(u);
    slope = x >= 0.0f ? inverse : e * inverse;
    return fmaxf(x, 0.0f) + fmaf(__builtin_amdgcn_logf(u), 0.693147180559945309f, e - (u - 1.0f));
}
__device__ __forceinline__ float softplus_f32(float x) {
    float slope;
    return softplus_f32(x, slope);
}

// Makes the wave wait here for the loads into v, and not later, behind stores that follow: loads and stores
// complete in order, and a wait for a load behind a store that a branch may have skipped waits for the store too.
template <typename T, int V>
__device__ __forceinline__ void arrive(Pack<T, V>& v) {
    constexpr int WORDS = (sizeof(T) * V + 3) / 4;
    if constexpr (sizeof(T) * V == 2) {
        unsigned short u;
        __builtin_memcpy(&u, &v.v, 2);
        unsigned w = u;
        asm volatile("" : "+v"(w));
        u = (unsigned short)w;
        __builtin_memcpy(&v.v, &u, 2);
    } else {
        unsigned w[WORDS];
        __builtin_memcpy(w, &v.v, WORDS * 4);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
        __builtin_memcpy(&v.v, w, WORDS * 4);
    }
}
__device__ __forceinline__ void arrive(float& v) { asm volatile("" : "+v"(v)); }

// Orders the LDS traffic of one wave: its lanes read what other lanes of it wrote.  The hardware
// runs a wave's LDS instructions in order; this keeps the compiler from moving them.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// a and b with their 32-lane halves (16-lane odd / even rows) exchanged and added: lanes of the
// lower half (even rows) get the sum of a over the pair of lanes, the others that of b.
__device__ __forceinline__ float halves_sum(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rows_sum(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float dpp_mov(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over four neighbouring lanes, in all of them.
__device__ __forceinline__ float quad_sum(float v) {
    v += dpp_mov<0xB1>(v);      // quad_perm [1,0,3,2]
    v += dpp_mov<0x4E>(v);      // quad_perm [2,3,0,1]
    return v;
}
// Sum over the 16 lanes of a row, in all of them.
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_mov<0x128>(v);     // row_ror:8
    v += dpp_mov<0x124>(v);     // row_ror:4
    v += dpp_mov<0x122>(v);     // row_ror:2
    v += dpp_mov<0x121>(v);     // row_ror:1
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    v = rows_sum(v, v);
    return halves_sum(v, v);
}

// Zeros in the rows of a matrix that belong to no utterance: those before off[0] and from off[utts] on (all, without
// utterances).  Workgroup `group` of `groups` takes every groups-th of them.
template <typename T>
__device__ __forceinline__ void clear_other_rows(const int64_t* off, int64_t utts, int64_t frames, void* to, int64_t ld,
                                                 int64_t width, int64_t group, int64_t groups) {
    const int64_t first = utts > 0 ? min(max(off[0], (int64_t)0), frames) : 0;
    const int64_t last = utts > 0 ? min(max(off[utts], first), frames) : 0;
    for (int64_t i = group; i < frames - (last - first); i += groups) {
        T* row = (T*)to + (i < first ? i : i + (last - first)) * ld;
        for (int64_t c = threadIdx.x; c < width; c += blockDim.x) row[c] = (T)0.0f;
    }
}
constexpr int kClearGroups = 64;        // workgroups behind a launch's own ones that do this: next to nothing if there is nothing to do

// Parts [parts][columns] added up in a fixed order, 32 columns a workgroup and every 32nd part a thread; `store` takes
// a column's sum.
constexpr int kSumThreads = 1024;
template <typename F>
__device__ __forceinline__ void sum_parts(const float* part, int64_t parts, int64_t columns, F store) {
    __shared__ double sums[32][33];
    const int at = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t column = (int64_t)blockIdx.x * 32 + at;
    double s = 0.0;
    if (column < columns) {
        int64_t k = slice;
        for (; k + 96 < parts; k += 128) {               // four loads in flight
            const float a = part[k * columns + column], b = part[(k + 32) * columns + column];
            const float c = part[(k + 64) * columns + column], d = part[(k + 96) * columns + column];
            s += ((double)a + (double)b) + ((double)c + (double)d);
        }
        for (; k < parts; k += 32) s += (double)part[k * columns + column];
    }
    sums[slice][at] = s;
    __syncthreads();
    if (slice != 0 || column >= columns) return;
    s = 0.0;
    for (int k = 0; k < 32; ++k) s += sums[k][at];
    store(column, s);
}

// Entry points run on the context's device and leave the caller's current device alone.
struct DeviceGuard {
    int before = -1, rc = SRX_OK;
    explicit DeviceGuard(int device) {
        rc = enter(device);
    }
    int enter(int device) {
        int now = -1;
        SRX_HIP(hipGetDevice(&now));
        if (now != device) {
            SRX_HIP(hipSetDevice(device));
            before = now;
        }
        return SRX_OK;
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;
};

constexpr int kMostColumns = 1 << 24;           // values of a row, so that 32 bits count them and what lies beside them
// Whether the caller wants zeros in y's rows of no utterance; leaves the element type.
inline bool take_zero_rows(int& dtype) {
    const bool zero = dtype >= 0 && (dtype & SRX_ZERO_OTHER_ROWS) != 0;
    if (zero) dtype &= ~SRX_ZERO_OTHER_ROWS;
    return zero;
}
inline bool frame_dtype(int dtype) { return dtype == SRX_F32 || dtype == SRX_BF16 || dtype == SRX_F16; }

}  // namespace srx_frames
