// Shared by the operators over packed rows (packed_conv.h, packed_scan.h, packed_norm.h):
// element types, wide loads at any element alignment, the place of a row in its sequence, wavefront
// sums, and the error convention of the C ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>
#include <string>
#include <type_traits>

#include "../../include/mfcc_hip.h"

namespace mfcc_detail {
int fail(int code, const char* msg);     // sets the thread-local message behind mfcc_last_error(); never throws
}

#define PACKED_CATCH_ALL                                                              \
    catch (const std::bad_alloc&) {                                                   \
        return mfcc_detail::fail(MFCC_E_NOMEM, "out of host memory");                 \
    } catch (...) {                                                                   \
        return mfcc_detail::fail(MFCC_E_INVALID, "unexpected C++ exception");         \
    }

#define PACKED_LAUNCHED()                                                             \
    do {                                                                              \
        const hipError_t e_ = hipGetLastError();                                      \
        if (e_ != hipSuccess) return mfcc_detail::fail(MFCC_E_HIP, hipGetErrorString(e_)); \
    } while (0)

namespace packed {

constexpr int WAVE = 64;

// ---- element types ---------------------------------------------------------------------------
// Every operator computes in float32; the 16-bit types exist in memory only.  The conversions to
// them round once, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32).
struct F32 { using mem = float; };
struct BF16 { using mem = __bf16; };
struct F16 { using mem = _Float16; };

template <typename M> __device__ __forceinline__ float widen(M v) { return (float)v; }
template <typename M> __device__ __forceinline__ M narrow(float v) { return (M)v; }

// VEC elements as they lie in memory, in 32-bit words: in the 16-bit types half the registers until they are used,
// and one wide access (an array of a 16-bit type takes a register, and often a load, per element: 166 instead of
// 98 us for the convolution of 30011 x 4096).
template <typename M, int VEC>
struct Raw {
    uint32_t u[VEC * sizeof(M) / 4];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(M) == 4) return __uint_as_float(u[i]);
        else if constexpr (std::is_same<M, __bf16>::value) return __uint_as_float(i % 2 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
        else return (float)__builtin_bit_cast(M, (uint16_t)(u[i / 2] >> (i % 2 * 16)));
    }
    __device__ __forceinline__ void set(const float (&v)[VEC]) {
        if constexpr (sizeof(M) == 4) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) u[i] = __float_as_uint(v[i]);
        } else {
            typedef float f2 __attribute__((ext_vector_type(2)));
            typedef M m2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int i = 0; i < VEC; i += 2) u[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[i], v[i + 1]}, m2));
        }
    }
};

// From and to an address that is only aligned to its element: global memory takes wide accesses at any such
// address on gfx950, so a row of any width and stride uses the same loads.  n < VEC (the ragged end of a row) goes
// element by element.
// Elements behind a row's last are read along with it where the tensor goes on behind the row (any row but the last,
// rows at least VEC - 1 apart) and thrown away: taking the last n < VEC one by one in a 16-bit type packs them where they
// are loaded, and so waits for every load in flight (gradients of the gated norm at 12001 x 1545 in bfloat16 54 instead of 48 us).
inline bool has_room(const void* p, int64_t stride, int vec) { return !p || stride >= vec - 1; }

template <typename M, int VEC>
__device__ __forceinline__ void load_raw(Raw<M, VEC>& v, const M* __restrict__ p, int n, bool room = false) {
    if (n >= VEC || (room && n > 0)) {
        __builtin_memcpy(v.u, p, sizeof(v.u));
    } else {
        float e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = i < n ? widen(p[i]) : 0.0f;
        v.set(e);
    }
}

template <typename M, int VEC>
__device__ __forceinline__ void load_vec(float (&v)[VEC], const M* __restrict__ p, int n, bool room = false) {
    Raw<M, VEC> raw;
    load_raw<M, VEC>(raw, p, n, room);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = raw.get(i);
}

template <typename M, int VEC>
__device__ __forceinline__ void store_vec(M* __restrict__ p, const float (&v)[VEC], int n) {
    if (n >= VEC) {
        Raw<M, VEC> raw;
        raw.set(v);
        __builtin_memcpy(p, raw.u, sizeof(raw.u));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < n) p[i] = narrow<M>(v[i]);
    }
}

// ---- functions ---------------------------------------------------------------------------------
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// exp(x) = exp2(p) exp(x - p ln 2) with p the rounded x log2(e): the second factor is 1 + (x - p ln 2) within 2^-36, and
// p ln 2 in two floats keeps the error from growing with |x| (at most two units beside exp2's own).
constexpr float LN2_REST = -1.90465429995776804525e-9f;       // ln 2 - LN2
__device__ __forceinline__ float exp_rest(float x, float p) { return fmaf(p, -LN2_REST, fmaf(p, -LN2, x)); }
__device__ __forceinline__ float exp_f(float x) {
    const float p = x * LOG2E, e = exp2_hw(p);
    // outside the finite, normal range the correction is meaningless (and inf * 0 or inf - inf appears in it)
    return fabsf(p) < 126.0f ? fmaf(e, exp_rest(x, p), e) : e;
}

__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.0f + exp_f(-x)); }

// For a result that is rounded to 16 bits and goes nowhere else: without the second float of the exponent's product
// the sigmoid is off by |x| 2^-24 more, below 2^-17 up to |x| = 88, where it leaves float32's range; half a step of
// bfloat16 is up to 2^-8 of the value, of float16 2^-11.  Whatever has float32 results takes sigmoid_f.
__device__ __forceinline__ float sigmoid_to_16(float x) { return rcp_hw(1.0f + exp2_hw(x * -LOG2E)); }

// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|) in (0, 1].  w = 1 + e loses the low bits of a
// small e; what it lost, e - (w - 1), is exact and is added back (to first order: the error of that is
// below 2^-24 e).
__device__ __forceinline__ float softplus_f(float x) {
    // exp_f of -|x|: the bound takes away the infinity and changes nothing else (exp(-100) is below float32's normal range)
    const float v = __builtin_elementwise_maximum(-fabsf(x), -100.0f);     // a NaN stays
    const float p = v * LOG2E, e0 = exp2_hw(p), e = fmaf(e0, exp_rest(v, p), e0);
    const float w = 1.0f + e;
    return fmaxf(x, 0.0f) + fmaf(log2_hw(w), LN2, e - (w - 1.0f));
}

// ---- where a row lies ----------------------------------------------------------------------------
// Sequence s holds the rows off[s] .. off[s + 1].  The offsets are device data that no host code has
// seen, so nothing read from them is trusted as an index: a row that is inside the sequence found for it
// satisfies 0 <= start <= row < end, and rows are never addressed outside [0, rows).
struct Place {
    int s;               // sequence, in [0, n_seqs)
    int64_t start, end;  // its rows (start <= row < end) when inside, clipped to [0, rows]
    int64_t until;       // first row at which this answer may change (> row)
    bool inside;
};

__device__ __forceinline__ Place find_row(const int64_t* __restrict__ off, int n_seqs, int64_t rows, int64_t row) {
    Place p;
    if (!off) {          // one sequence of all rows
        p.s = 0; p.start = 0; p.end = rows; p.until = rows; p.inside = row < rows;
        return p;
    }
    int lo = 0, hi = n_seqs;                    // the last s with off[s] <= row, or 0
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= row) lo = mid; else hi = mid;
    }
    p.s = lo;
    p.start = off[lo];
    p.end = min(off[lo + 1], rows);
    p.inside = p.start >= 0 && p.start <= row && row < p.end;
    if (p.inside) p.until = p.end;
    else if (row < p.start) p.until = min(p.start, rows);          // before the first sequence
    else if (lo == n_seqs - 1) p.until = rows;                     // behind the last one
    else p.until = row + 1;                                        // offsets that do not ascend
    return p;
}

// A value that is the same in all lanes, in a scalar register -- and, through the empty asm, known as such to
// the compiler, which otherwise keeps loop counters that come out of a search in vector registers and
// computes addresses and branches from them lane by lane.
__device__ __forceinline__ int uniform(int v) {
    v = __builtin_amdgcn_readfirstlane(v);
    asm("" : "+s"(v));
    return v;
}

// The same for a whole wavefront, in scalar registers and relative to row r0 of a piece of `len` rows: which
// rows from t on lie in one sequence (or in none), and what happens at their ends.
struct Stretch {
    int s;               // sequence
    int until;           // first row (<= len) at which the answer may change
    int inside, first, last;    // in a sequence; row t is its first row; row until - 1 is its last one
};

__device__ __forceinline__ Stretch find_stretch(const int64_t* __restrict__ off, int n_seqs, int64_t rows, int64_t r0, int t,
                                                int len) {
    const Place p = find_row(off, n_seqs, rows, r0 + t);
    Stretch w;
    w.s = uniform(p.s);
    w.until = uniform((int)min(p.until - r0, (int64_t)len));
    const int flags = uniform((p.inside ? 1 : 0) | (p.start == r0 + t ? 2 : 0) | (p.end - r0 <= len ? 4 : 0));
    w.inside = flags & 1;
    w.first = flags & 2;
    w.last = (flags & 5) == 5 ? 1 : 0;
    return w;
}

// ---- wavefront helpers ----------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// lanes 0..31: x summed with its upper half; lanes 32..63: y summed with its lower half
__device__ __forceinline__ float halve32(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// even rows of 16 lanes: x summed over the pair of rows; odd rows: y
__device__ __forceinline__ float halve16(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over 16, 32 or (any larger COUNT) 64 neighbouring lanes, in every one of them.
template <int COUNT>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<0xB1>(v);          // quad_perm [1, 0, 3, 2]
    v += dpp<0x4E>(v);          // quad_perm [2, 3, 0, 1]
    v += dpp<0x141>(v);         // row_half_mirror
    v += dpp<0x140>(v);         // row_mirror
    if (COUNT >= 32) v = halve16(v, v);
    if (COUNT >= 64) v = halve32(v, v);
    return v;
}

// Whether another entry of a batch names the slot of entry e0 + k, before or after it.  The four wavefronts of the
// workgroup share the list; a short one each looks through by itself.
template <int NE>
__device__ __forceinline__ void slot_use(bool (&before)[NE], bool (&after)[NE], const int32_t* __restrict__ slots, int batch,
                                         int e0, const int (&slot)[NE]) {
    __shared__ unsigned found[4];
    const bool alone = batch <= WAVE;
    unsigned bits = 0;
#pragma unroll 4
    for (int e = alone ? threadIdx.x & 63 : threadIdx.x; e < batch; e += 256) {
        const int other = slots[e];
#pragma unroll
        for (int k = 0; k < NE; ++k)
            if (other == slot[k]) bits |= (e < e0 + k ? 1u : e > e0 + k ? 16u : 0u) << k;
    }
    unsigned all = 0;
#pragma unroll
    for (int k = 0; k < NE; ++k) all |= (__ballot(bits >> k & 1) ? 1u << k : 0u) | (__ballot(bits >> k & 16) ? 16u << k : 0u);
    if (!alone) {
        if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = all;
        __syncthreads();
        all = found[0] | found[1] | found[2] | found[3];
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) { before[k] = all >> k & 1; after[k] = all >> k & 16; }
}

// Workgroups are dealt to the eight XCDs in turn.  This gives each XCD a contiguous eighth of the work, so that
// neighbouring pieces, which share rows, share an L2.
__device__ __forceinline__ unsigned xcd_order(unsigned block, unsigned blocks) {
    const unsigned each = blocks / 8, rest = blocks % 8, xcd = block % 8;
    return xcd * each + min(xcd, rest) + block / 8;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// p[first] + p[first + step] + ... of `count` terms `stride` apart, eight loads in flight; a fixed order.
__device__ __forceinline__ float sum_strided(const float* __restrict__ p, int64_t first, int64_t step, int64_t count,
                                             int64_t stride) {
    float s = 0.0f;
    int64_t i = first;
    for (; i + 7 * step < count; i += 8 * step) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[(i + j * step) * stride];
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; i < count; i += step) s += p[i * stride];
    return s;
}

template <typename Fn>
int by_type(int dtype, Fn&& fn) {
    switch (dtype) {
        case MFCC_F32: return fn(F32{});
        case MFCC_BF16: return fn(BF16{});
        case MFCC_F16: return fn(F16{});
    }
    return mfcc_detail::fail(MFCC_E_INVALID, "unknown element type");
}

}  // namespace packed
