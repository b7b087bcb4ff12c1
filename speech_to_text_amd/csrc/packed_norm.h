// Norms before and after a block, fused with the residual sum and its scale, or with the gate.
//   add:   r = residual + scale x;  y = norm(r) w + b
//   gate:  y = norm(x silu(z)) w + b  or  (norm(x) w + b) silu(z), over `groups` slices of the row
//   norm:  v / sqrt(mean(v^2) + eps), of v - mean(v) for the layer form.
// Bound by memory: every row is read once, held in registers (eight neighbouring elements a thread and
// step), reduced over 64, 256 or 1024 threads and written once.  The layer form's deviation is summed
// around the mean, from the registers.
#pragma once
#include "packed.h"

namespace packed {

constexpr int NV = 8;

struct Norm {
    const void *x, *z, *residual, *r_in, *dy, *dr;
    int64_t x_stride, z_stride, residual_stride, r_stride, y_stride, dy_stride, dr_stride;
    const float *weight, *bias, *scale;
    void *y, *r, *dx, *dz, *dresidual;
    float* part;               // (blocks, 3, channels): dweight, dbias, dscale
    int64_t rows;
    int channels, groups, width, layer, gate_first;
    float eps, scale_value, inv_width;
};

// Sums of two values over the TPU threads of a unit.
template <int TPU>
__device__ __forceinline__ void unit_sum2(float& a, float& b, float (*sh)[2]) {
    a = wave_sum(a); b = wave_sum(b);
    if (TPU > WAVE) {
        constexpr int W = TPU / WAVE;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { sh[wave][0] = a; sh[wave][1] = b; }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) { a += sh[w][0]; b += sh[w][1]; }
    }
}

template <typename M>
__device__ __forceinline__ void load_or(float (&v)[NV], const M* p, int n, float other) {
    if (p) load_vec<M, NV>(v, p, n);
    else {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = other;
    }
}

template <typename T, typename RT, bool GATE, int TPU, int IT>
__global__ __launch_bounds__(TPU < 256 ? 256 : TPU) void k_norm_fwd(const Norm a) {
    using M = typename T::mem;
    using RM = typename RT::mem;
    constexpr int PER = TPU < 256 ? 256 / TPU : 1;
    __shared__ float sh[TPU > WAVE ? TPU / WAVE : 1][2];
    const int64_t unit = (int64_t)blockIdx.x * PER + (PER > 1 ? threadIdx.x / TPU : 0);
    if (unit >= a.rows * a.groups) return;                    // whole wavefronts of a one-wavefront unit
    const int64_t row = a.groups > 1 ? unit / a.groups : unit;
    const int c_base = a.groups > 1 ? (int)(unit % a.groups) * a.width : 0;
    const int tid = PER > 1 ? threadIdx.x % TPU : threadIdx.x;
    const M* x = static_cast<const M*>(a.x) + row * a.x_stride;

    float v[IT][NV], gate[GATE ? IT : 1][NV], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int w0 = (k * TPU + tid) * NV, c = c_base + w0, n = max(a.width - w0, 0);
        float xv[NV];
        load_vec<M, NV>(xv, x + c, n);
        if (GATE) {
            load_vec<M, NV>(gate[k], static_cast<const M*>(a.z) + row * a.z_stride + c, n);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                gate[k][i] *= sigmoid_f(gate[k][i]);
                v[k][i] = a.gate_first ? xv[i] * gate[k][i] : xv[i];
            }
        } else {
            float sc[NV], rv[NV];
            load_or<float>(sc, a.scale ? a.scale + c : nullptr, n, a.scale_value);
            load_or<RM>(rv, a.residual ? static_cast<const RM*>(a.residual) + row * a.residual_stride + c : nullptr, n, 0.0f);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[k][i] = fmaf(sc[i], xv[i], rv[i]);
            if (n < NV) {
#pragma unroll
                for (int i = 0; i < NV; ++i) v[k][i] = i < n ? v[k][i] : 0.0f;
            }
            if (a.r && n > 0) store_vec<RM, NV>(static_cast<RM*>(a.r) + row * a.r_stride + c, v[k], n);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) { s1 += v[k][i]; s2 = fmaf(v[k][i], v[k][i], s2); }
    }
    unit_sum2<TPU>(s1, s2, sh);
    float mean = 0.0f;
    if (a.layer) {
        mean = s1 * a.inv_width;
        s1 = s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int n = a.width - (k * TPU + tid) * NV;
#pragma unroll
            for (int i = 0; i < NV; ++i) { const float d = i < n ? v[k][i] - mean : 0.0f; s2 = fmaf(d, d, s2); }
        }
        unit_sum2<TPU>(s1, s2, sh);
    }
    const float q = rsqrtf(fmaf(s2, a.inv_width, a.eps));
    M* y = static_cast<M*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int w0 = (k * TPU + tid) * NV, c = c_base + w0, n = a.width - w0;
        if (n <= 0) continue;
        float w[NV], b[NV];
        load_or<float>(w, a.weight ? a.weight + c : nullptr, n, 1.0f);
        load_or<float>(b, a.bias ? a.bias + c : nullptr, n, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o = fmaf((v[k][i] - mean) * q, w[i], b[i]);
            if (GATE && !a.gate_first) o *= gate[k][i];
            v[k][i] = o;
        }
        store_vec<M, NV>(y + c, v[k], n);
    }
}

// A block keeps its columns and walks over rows; the sums over rows stay in registers until its end, then
// one partial row per block is written and k_norm_reduce adds those in a fixed order.
template <typename T, typename RT, bool GATE, int TPU, int IT>
__global__ __launch_bounds__(TPU < 256 ? 256 : TPU) void k_norm_bwd(const Norm a) {
    using M = typename T::mem;
    using RM = typename RT::mem;
    constexpr int PER = TPU < 256 ? 256 / TPU : 1;
    __shared__ float sh[TPU > WAVE ? TPU / WAVE : 1][2];
    __shared__ float fold[PER > 1 ? PER : 1][PER > 1 ? TPU * NV : 1];
    const int slot = PER > 1 ? threadIdx.x / TPU : 0, tid = PER > 1 ? threadIdx.x % TPU : threadIdx.x;
    const int c_base = blockIdx.y * a.width;
    float dw[IT][NV] = {}, db[IT][NV] = {}, ds[GATE ? 1 : IT][NV] = {};

    for (int64_t row = (int64_t)blockIdx.x * PER + slot; row < a.rows; row += (int64_t)gridDim.x * PER) {
        float v[IT][NV], dn[IT][NV], s1 = 0.0f, s2 = 0.0f, t1 = 0.0f, t2 = 0.0f;
        float xv[IT][NV], zv[GATE ? IT : 1][NV], dyv[IT][NV];
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int w0 = (k * TPU + tid) * NV, c = c_base + w0, n = max(a.width - w0, 0);
            load_or<M>(dyv[k], a.dy ? static_cast<const M*>(a.dy) + row * a.dy_stride + c : nullptr, n, 0.0f);
            float w[NV];
            load_or<float>(w, a.weight ? a.weight + c : nullptr, n, 1.0f);
            if (GATE) {
                load_vec<M, NV>(xv[k], static_cast<const M*>(a.x) + row * a.x_stride + c, n);
                load_vec<M, NV>(zv[k], static_cast<const M*>(a.z) + row * a.z_stride + c, n);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float gate = zv[k][i] * sigmoid_f(zv[k][i]);
                    v[k][i] = a.gate_first ? xv[k][i] * gate : xv[k][i];
                    dn[k][i] = (a.gate_first ? dyv[k][i] : dyv[k][i] * gate) * w[i];
                }
            } else {
                load_vec<RM, NV>(v[k], static_cast<const RM*>(a.r_in) + row * a.r_stride + c, n);
#pragma unroll
                for (int i = 0; i < NV; ++i) dn[k][i] = dyv[k][i] * w[i];
            }
            if (n < NV) {
#pragma unroll
                for (int i = 0; i < NV; ++i) { dn[k][i] = i < n ? dn[k][i] : 0.0f; v[k][i] = i < n ? v[k][i] : 0.0f; }
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s1 += v[k][i]; t1 += dn[k][i];
                s2 = fmaf(v[k][i], v[k][i], s2); t2 = fmaf(dn[k][i], v[k][i], t2);
            }
        }
        float mean = 0.0f, dmean = 0.0f;
        if (a.layer) {
            unit_sum2<TPU>(s1, t1, sh);
            mean = s1 * a.inv_width; dmean = t1 * a.inv_width;
            s2 = t2 = 0.0f;
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int n = a.width - (k * TPU + tid) * NV;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float d = i < n ? v[k][i] - mean : 0.0f;
                    v[k][i] = d;
                    s2 = fmaf(d, d, s2); t2 = fmaf(dn[k][i], d, t2);
                }
            }
        }
        unit_sum2<TPU>(s2, t2, sh);
        const float q = rsqrtf(fmaf(s2, a.inv_width, a.eps));
        const float proj = t2 * a.inv_width * q;                 // mean(dn * v q)
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int w0 = (k * TPU + tid) * NV, c = c_base + w0, n = a.width - w0;
            if (n <= 0) continue;
            float dv[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float vn = v[k][i] * q;
                dv[i] = (dn[k][i] - dmean - vn * proj) * q;
                v[k][i] = vn;
            }
            const int64_t at = row * a.channels + c;
            if (GATE) {
                float dz[NV], w[NV], b[NV];
                load_or<float>(w, a.weight ? a.weight + c : nullptr, n, 1.0f);
                load_or<float>(b, a.bias ? a.bias + c : nullptr, n, 0.0f);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float z = zv[k][i], sg = sigmoid_f(z), gate = z * sg, slope = sg * fmaf(z, 1.0f - sg, 1.0f);
                    const float body = a.gate_first ? dyv[k][i] : dyv[k][i] * gate;
                    dz[i] = (a.gate_first ? dv[i] * xv[k][i] : dyv[k][i] * fmaf(v[k][i], w[i], b[i])) * slope;
                    if (a.gate_first) dv[i] *= gate;
                    dw[k][i] = fmaf(body, v[k][i], dw[k][i]);
                    db[k][i] += body;
                }
                store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                store_vec<M, NV>(static_cast<M*>(a.dz) + at, dz, n);
            } else {
                float dr[NV];
                load_or<RM>(dr, a.dr ? static_cast<const RM*>(a.dr) + row * a.dr_stride + c : nullptr, n, 0.0f);
                if (a.x) load_vec<M, NV>(xv[k], static_cast<const M*>(a.x) + row * a.x_stride + c, n);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    dv[i] += dr[i];
                    dw[k][i] = fmaf(dyv[k][i], v[k][i], dw[k][i]);
                    db[k][i] += dyv[k][i];
                    if (a.x) ds[k][i] = fmaf(dv[i], xv[k][i], ds[k][i]);
                }
                if (a.dresidual) store_vec<RM, NV>(static_cast<RM*>(a.dresidual) + at, dv, n);
                if (a.dx) {
                    float sc[NV];
                    load_or<float>(sc, a.scale ? a.scale + c : nullptr, n, a.scale_value);
#pragma unroll
                    for (int i = 0; i < NV; ++i) dv[i] *= sc[i];
                    store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                }
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < (GATE ? 2 : 3); ++j) {
        float* out = a.part + ((int64_t)blockIdx.x * 3 + j) * a.channels + c_base;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const float (&s)[NV] = j == 0 ? dw[k] : j == 1 ? db[k] : ds[GATE ? 0 : k];
            const int w0 = (k * TPU + tid) * NV;
            if (PER > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NV; ++i) fold[slot][i * TPU + tid] = s[i];
                __syncthreads();
                for (int e = threadIdx.x; e < TPU * NV; e += 256) {
                    float t = 0.0f;
#pragma unroll
                    for (int p = 0; p < PER; ++p) t += fold[p][(e % NV) * TPU + e / NV];
                    if (k * TPU * NV + e < a.width) out[k * TPU * NV + e] = t;
                }
            } else if (w0 < a.width) {
                store_vec<float, NV>(out + w0, s, a.width - w0);
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_reduce(const float* __restrict__ part, int n_part, int channels, float* dweight,
                                                      float* dbias, float* dscale) {
    __shared__ float sh[16][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, j = blockIdx.y;
    float* out = j == 0 ? dweight : j == 1 ? dbias : dscale;
    if (!out) return;
    sh[slice][lane] = c < channels ? sum_strided(part + (int64_t)j * channels + c, slice, 16, n_part, 3 * (int64_t)channels) : 0.0f;
    __syncthreads();
    if (slice == 0 && c < channels) {
        float t = 0.0f;
#pragma unroll
        for (int p = 0; p < 16; ++p) t += sh[p][lane];
        out[c] = t;
    }
}

// ---- host --------------------------------------------------------------------------------------------
constexpr int NORM_MAX_WIDTH = 32768;

// Threads per row and steps of eight elements per thread: (64, 1) .. (1024, 4).
template <typename Fn>
int by_width_of_row(int width, Fn&& fn) {
    using std::integral_constant;
    if (width <= 512) return fn(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (width <= 2048) return fn(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (width <= 4096) return fn(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (width <= 8192) return fn(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
    if (width <= 16384) return fn(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    return fn(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
}

// Blocks that walk over the rows in the backward pass: four of 256 threads for each of the 256 CUs.
inline int norm_bwd_blocks(const mfcc_norm_args* a) {
    const int width = a->channels / a->groups, per = width <= 512 ? 4 : 1;
    const int64_t most = std::max<int64_t>(1, (width <= 4096 ? 1024 : 512) / a->groups);
    return (int)std::min<int64_t>(ceil_div(a->rows, per), most);
}

inline Norm norm_args(const mfcc_norm_args* a) {
    Norm f = {};
    f.x = a->d_x; f.z = a->d_z; f.residual = a->d_residual; f.r_in = a->d_r; f.dy = a->d_dy; f.dr = a->d_dr;
    f.x_stride = a->x_stride; f.z_stride = a->z_stride; f.residual_stride = a->residual_stride; f.r_stride = a->r_stride;
    f.y_stride = a->y_stride; f.dy_stride = a->dy_stride; f.dr_stride = a->dr_stride;
    f.weight = a->d_weight; f.bias = a->d_bias; f.scale = a->d_scale; f.y = a->d_y; f.r = a->d_r; f.dx = a->d_dx;
    f.dz = a->d_dz; f.dresidual = a->d_dresidual; f.rows = a->rows; f.channels = a->channels; f.groups = a->groups;
    f.width = a->channels / a->groups; f.layer = a->norm == MFCC_NORM_LAYER; f.gate_first = a->gate_first;
    f.eps = a->eps; f.scale_value = a->scale_value; f.inv_width = 1.0f / (float)f.width;
    return f;
}

template <typename T, typename RT, bool GATE>
int norm_forward(const mfcc_norm_args* a, hipStream_t st) {
    if (a->rows == 0) return MFCC_OK;
    const Norm f = norm_args(a);
    return by_width_of_row(f.width, [&](auto tpu, auto it) {
        constexpr int TPU = decltype(tpu)::value, IT = decltype(it)::value, PER = TPU < 256 ? 256 / TPU : 1;
        const int64_t blocks = ceil_div(f.rows * f.groups, PER);
        if (blocks > 0x3fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
        hipLaunchKernelGGL((k_norm_fwd<T, RT, GATE, TPU, IT>), dim3((unsigned)blocks), dim3(TPU < 256 ? 256 : TPU), 0, st, f);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

template <typename T, typename RT, bool GATE>
int norm_backward(const mfcc_norm_args* a, hipStream_t st) {
    Norm f = norm_args(a);
    if (!a->d_dscale && !GATE) f.x = nullptr;
    const int blocks = norm_bwd_blocks(a);
    const bool sums = a->d_dweight || a->d_dbias || a->d_dscale;
    f.part = sums ? static_cast<float*>(a->d_workspace) : nullptr;
    return by_width_of_row(f.width, [&](auto tpu, auto it) {
        constexpr int TPU = decltype(tpu)::value, IT = decltype(it)::value;
        if (blocks > 0) {
            hipLaunchKernelGGL((k_norm_bwd<T, RT, GATE, TPU, IT>), dim3((unsigned)blocks, (unsigned)f.groups),
                               dim3(TPU < 256 ? 256 : TPU), 0, st, f);
            PACKED_LAUNCHED();
        }
        if (sums) {
            hipLaunchKernelGGL(k_norm_reduce<T>, dim3((unsigned)ceil_div(f.channels, 64), 3), dim3(1024), 0, st, f.part, blocks,
                               f.channels, a->d_dweight, a->d_dbias, a->d_dscale);
            PACKED_LAUNCHED();
        }
        return (int)MFCC_OK;
    });
}

template <typename T>
int add_norm_forward(const mfcc_norm_args* a, hipStream_t st) {
    return a->res_dtype == a->dtype ? norm_forward<T, T, false>(a, st) : norm_forward<T, F32, false>(a, st);
}
template <typename T>
int add_norm_backward(const mfcc_norm_args* a, hipStream_t st) {
    return a->res_dtype == a->dtype ? norm_backward<T, T, false>(a, st) : norm_backward<T, F32, false>(a, st);
}
template <typename T>
int gate_norm_forward(const mfcc_norm_args* a, hipStream_t st) { return norm_forward<T, T, true>(a, st); }
template <typename T>
int gate_norm_backward(const mfcc_norm_args* a, hipStream_t st) { return norm_backward<T, T, true>(a, st); }

}  // namespace packed
