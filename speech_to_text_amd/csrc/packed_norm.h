// Norms before and after a block, fused with the residual sum and its scale, or with the gate.
//   add:   r = residual + scale x;  y = norm(r) w + b
//   gate:  y = norm(x silu(z)) w + b  or  (norm(x) w + b) silu(z), over `groups` slices of the row
//   norm:  v / sqrt(mean(v^2) + eps), of v - mean(v) for the layer form.
// Bound by memory: every row is read once, held in registers (eight neighbouring elements a thread and
// step), reduced over 16 to 1024 threads and written once.  The layer form's deviation is summed
// around the mean, from the registers.  16384 x 2048, bfloat16 with a float32 residual: 82 us forward (4.9 TB/s), 118 us
// backward (5.1 TB/s); the gate over 30011 x 4096 in 8 groups, bfloat16: 136 us (5.4 TB/s, two reads to a write).
#pragma once
#include "packed.h"

namespace packed {

constexpr int NV = 8;

// Threads of a workgroup: several rows within wavefronts, or one row of several wavefronts.
constexpr int norm_block(int threads_per_row) { return threads_per_row <= WAVE ? 256 : threads_per_row; }

struct Norm {
    const void *x, *z, *residual, *r_in, *dy, *dr;
    int64_t x_stride, z_stride, residual_stride, r_stride, y_stride, dy_stride, dr_stride;
    const float *weight, *bias, *scale;
    void *y, *r, *dx, *dz, *dresidual;
    float* part;               // (blocks, 3, channels): dweight, dbias, dscale
    float4* stats;             // wide rows: mean, 1 / deviation, and their gradient's (rows, groups)
    int64_t rows;
    int channels, groups, width, layer, gate_first, room;
    bool want[3];              // of the three sums
    float eps, scale_value, inv_width;
};

// Sums of two values over the TPU threads of a unit.
template <int TPU>
__device__ __forceinline__ void unit_sum2(float& a, float& b, float (*sh)[2]) {
    a = lanes_sum<TPU>(a); b = lanes_sum<TPU>(b);
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
__device__ __forceinline__ void load_or(float (&v)[NV], const M* p, int n, float other, bool room = false) {
    if (p) load_vec<M, NV>(v, p, n, room);
    else {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = other;
    }
}

template <typename T, typename RT, bool GATE, int TPU, int IT>
__global__ __launch_bounds__(norm_block(TPU)) void k_norm_fwd(const Norm a) {
    using M = typename T::mem;
    using RM = typename RT::mem;
    constexpr int PER = norm_block(TPU) / TPU;
    __shared__ float sh[TPU > WAVE ? TPU / WAVE : 1][2];
    const int64_t unit = (int64_t)blockIdx.x * PER + (PER > 1 ? threadIdx.x / TPU : 0);
    if (unit >= a.rows * a.groups) return;                    // the sums of a smaller unit stay in its own lanes
    const int64_t row = a.groups > 1 ? unit / a.groups : unit;
    const int c_base = a.groups > 1 ? (int)(unit % a.groups) * a.width : 0;
    const int tid = PER > 1 ? threadIdx.x % TPU : threadIdx.x;
    const M* x = static_cast<const M*>(a.x) + row * a.x_stride;

    float v[IT][NV], gate[GATE ? IT : 1][NV], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int w0 = (k * TPU + tid) * NV, c = c_base + w0, n = max(a.width - w0, 0);
        const bool room = a.room && row + 1 < a.rows;
        float xv[NV];
        load_vec<M, NV>(xv, x + c, n, room);
        if (GATE) {
            load_vec<M, NV>(gate[k], static_cast<const M*>(a.z) + row * a.z_stride + c, n, room);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                gate[k][i] *= sigmoid_f(gate[k][i]);
                v[k][i] = a.gate_first ? xv[i] * gate[k][i] : xv[i];
            }
        } else {
            float sc[NV], rv[NV];
            load_or<float>(sc, a.scale ? a.scale + c : nullptr, n, a.scale_value);
            load_or<RM>(rv, a.residual ? static_cast<const RM*>(a.residual) + row * a.residual_stride + c : nullptr, n, 0.0f, room);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[k][i] = fmaf(sc[i], xv[i], rv[i]);
        }
        if (n < NV) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[k][i] = i < n ? v[k][i] : 0.0f;
        }
        if (!GATE) {
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
// one partial row per block is written and k_norm_reduce adds those in a fixed order.  With eight elements a thread
// (IT = 1) the tables stay in registers and the next row is in flight during the reductions of the current one (for
// the gate in 16-bit types only: three float32 rows ahead cost a wavefront per SIMD, 28 against 26 us at 4099 x 1537).
// Four wavefronts per SIMD in 16-bit types, a few registers spilled: the gate at 16384 x 2048 83 -> 72 us.
template <typename T, int IT> constexpr int norm_bwd_waves() { return IT == 1 && sizeof(typename T::mem) == 2 ? 4 : 1; }
template <typename T, typename RT, bool GATE, int TPU, int IT>
__global__ __launch_bounds__(norm_block(TPU)) __attribute__((amdgpu_waves_per_eu(norm_bwd_waves<T, IT>())))
void k_norm_bwd(const Norm a) {
    using M = typename T::mem;
    using RM = typename RT::mem;
    constexpr int PER = norm_block(TPU) / TPU;
    constexpr bool HELD = IT == 1, AHEAD_ROW = HELD && (!GATE || sizeof(M) == 2);
    __shared__ float sh[TPU > WAVE ? TPU / WAVE : 1][2];
    __shared__ float fold[PER > 1 ? PER : 1][PER > 1 ? TPU * NV : 1];
    const int slot = PER > 1 ? threadIdx.x / TPU : 0, tid = PER > 1 ? threadIdx.x % TPU : threadIdx.x;
    const int c_base = blockIdx.y * a.width;
    float dw[IT][NV] = {}, db[IT][NV] = {}, ds[GATE ? 1 : IT][NV] = {};
    auto left = [&](int k) { return max(a.width - (k * TPU + tid) * NV, 0); };
    auto col = [&](int k) { return c_base + (k * TPU + tid) * NV; };

    // what a row is made of: dy, and x and z (gate) or r, dr and x (add)
    struct RowIn { Raw<M, NV> dy[IT], x[IT], z[GATE ? IT : 1]; Raw<RM, NV> r[GATE ? 1 : IT], dr[GATE ? 1 : IT]; };
    auto fetch = [&](RowIn& in, int64_t row) {
        const float zero[NV] = {};
        const bool room = a.room && row + 1 < a.rows;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int c = col(k), all = left(k);
            auto take = [&](int n) {
                if (a.dy) load_raw<M, NV>(in.dy[k], static_cast<const M*>(a.dy) + row * a.dy_stride + c, n);
                else in.dy[k].set(zero);
                if (GATE || a.x) load_raw<M, NV>(in.x[k], static_cast<const M*>(a.x) + row * a.x_stride + c, n);
                if (GATE) {
                    load_raw<M, NV>(in.z[GATE ? k : 0], static_cast<const M*>(a.z) + row * a.z_stride + c, n);
                } else {
                    load_raw<RM, NV>(in.r[GATE ? 0 : k], static_cast<const RM*>(a.r_in) + row * a.r_stride + c, n);
                    if (a.dr) load_raw<RM, NV>(in.dr[GATE ? 0 : k], static_cast<const RM*>(a.dr) + row * a.dr_stride + c, n);
                    else in.dr[GATE ? 0 : k].set(zero);
                }
            };
            if (all >= NV || (room && all > 0)) take(NV);
            else take(all);
        }
    };
    // weight, and the bias (gate) or the scale (add)
    float w[IT][NV], t[IT][NV];
    auto tables = [&]() {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int c = col(k), n = left(k);
            load_or<float>(w[k], a.weight ? a.weight + c : nullptr, n, 1.0f);
            if (GATE) load_or<float>(t[k], a.bias ? a.bias + c : nullptr, n, 0.0f);
            else load_or<float>(t[k], a.scale ? a.scale + c : nullptr, n, a.scale_value);
        }
    };
    if (HELD) tables();

    const int64_t step = (int64_t)gridDim.x * PER;
    int64_t row = (int64_t)blockIdx.x * PER + slot;
    RowIn next;
    if (AHEAD_ROW && row < a.rows) fetch(next, row);
    for (; row < a.rows; row += step) {
        RowIn in;
        if (AHEAD_ROW) {
            in = next;
            if (row + step < a.rows) fetch(next, row + step);
        } else {
            fetch(in, row);
            if (!HELD) tables();
        }
        float v[IT][NV], dn[IT][NV], s1 = 0.0f, s2 = 0.0f, t1 = 0.0f, t2 = 0.0f;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int n = left(k);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float dy = in.dy[k].get(i);
                if (GATE) {
                    const float z = in.z[GATE ? k : 0].get(i), x = in.x[k].get(i), gate = z * sigmoid_f(z);
                    v[k][i] = a.gate_first ? x * gate : x;
                    dn[k][i] = (a.gate_first ? dy : dy * gate) * w[k][i];
                } else {
                    v[k][i] = in.r[GATE ? 0 : k].get(i);
                    dn[k][i] = dy * w[k][i];
                }
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
                const int n = left(k);
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
            const int c = col(k), n = left(k);
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
                float dz[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float z = in.z[GATE ? k : 0].get(i), x = in.x[k].get(i), dy = in.dy[k].get(i);
                    const float sg = sigmoid_f(z), gate = z * sg, slope = sg * fmaf(z, 1.0f - sg, 1.0f);
                    const float body = a.gate_first ? dy : dy * gate;
                    dz[i] = (a.gate_first ? dv[i] * x : dy * fmaf(v[k][i], w[k][i], t[k][i])) * slope;
                    if (a.gate_first) dv[i] *= gate;
                    dw[k][i] = fmaf(body, v[k][i], dw[k][i]);
                    db[k][i] += body;
                }
                store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                store_vec<M, NV>(static_cast<M*>(a.dz) + at, dz, n);
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float dy = in.dy[k].get(i);
                    dv[i] += in.dr[GATE ? 0 : k].get(i);
                    dw[k][i] = fmaf(dy, v[k][i], dw[k][i]);
                    db[k][i] += dy;
                }
                if (a.x) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) ds[GATE ? 0 : k][i] = fmaf(dv[i], in.x[k].get(i), ds[GATE ? 0 : k][i]);
                }
                if (a.dresidual) store_vec<RM, NV>(static_cast<RM*>(a.dresidual) + at, dv, n);
                if (a.dx) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) dv[i] *= t[k][i];
                    store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                }
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < (GATE ? 2 : 3); ++j) {
        if (!a.want[j]) continue;
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
                    float f = 0.0f;
#pragma unroll
                    for (int p = 0; p < PER; ++p) f += fold[p][(e % NV) * TPU + e / NV];
                    if (e < a.width) out[e] = f;
                }
            } else if (w0 < a.width) {
                store_vec<float, NV>(out + w0, s, a.width - w0);
            }
        }
    }
}

// ---- gradients of wide rows ----------------------------------------------------------------------------
// A row wider than the registers of a workgroup hold is read twice (three times for the layer form, whose deviation
// is summed around the mean), the second time from a cache.  The sums over rows are left to k_norm_columns, which
// reads everything once more with a thread per eight columns and takes the row's statistics from the workspace.
// Bound by memory: 1000 x 32768 in 104 us in bfloat16 and 237 us in float32 (2.5 and 2.2 TB/s of the residual norm's four
// tensors, those that are read twice counted once); the gate 130 and 288 us.

// Eight columns of a row.
template <typename T, typename RT, bool GATE>
struct NormColumns {
    float dy[NV], x[NV], z[NV], r[NV], dr[NV], w[NV], t[NV];
    __device__ __forceinline__ void tables(const Norm& a, int c, int n) {
        load_or<float>(w, a.weight ? a.weight + c : nullptr, n, 1.0f);
        if (GATE) load_or<float>(t, a.bias ? a.bias + c : nullptr, n, 0.0f);
        else load_or<float>(t, a.scale ? a.scale + c : nullptr, n, a.scale_value);
    }
    __device__ __forceinline__ void row(const Norm& a, int64_t row, int c, int n, bool all) {
        using M = typename T::mem;
        using RM = typename RT::mem;
        load_or<M>(dy, a.dy ? static_cast<const M*>(a.dy) + row * a.dy_stride + c : nullptr, n, 0.0f);
        if (GATE) {
            load_vec<M, NV>(x, static_cast<const M*>(a.x) + row * a.x_stride + c, n);
            load_vec<M, NV>(z, static_cast<const M*>(a.z) + row * a.z_stride + c, n);
        } else {
            load_vec<RM, NV>(r, static_cast<const RM*>(a.r_in) + row * a.r_stride + c, n);
            if (!all) return;
            load_or<RM>(dr, a.dr ? static_cast<const RM*>(a.dr) + row * a.dr_stride + c : nullptr, n, 0.0f);
            load_or<M>(x, a.x ? static_cast<const M*>(a.x) + row * a.x_stride + c : nullptr, n, 0.0f);
        }
    }
    __device__ __forceinline__ float gate(int i) const { return z[i] * sigmoid_f(z[i]); }
    // the value that is normalised, and the gradient of the normalised one
    __device__ __forceinline__ float value(const Norm& a, int i) const { return !GATE ? r[i] : a.gate_first ? x[i] * gate(i) : x[i]; }
    __device__ __forceinline__ float grad(const Norm& a, int i) const {
        return (GATE && !a.gate_first ? dy[i] * gate(i) : dy[i]) * w[i];
    }
};

template <typename T, typename RT, bool GATE>
__global__ __launch_bounds__(1024) void k_norm_bwd_wide(const Norm a) {
    using M = typename T::mem;
    using RM = typename RT::mem;
    __shared__ float sh[16][2];
    for (int64_t unit = blockIdx.x; unit < a.rows * a.groups; unit += gridDim.x) {
        const int64_t row = unit / a.groups;
        const int c_base = (int)(unit % a.groups) * a.width;
        NormColumns<T, RT, GATE> in;
        float mean = 0.0f, dmean = 0.0f, s = 0.0f, t = 0.0f;
        if (a.layer) {
            for (int w0 = threadIdx.x * NV; w0 < a.width; w0 += 1024 * NV) {
                const int n = a.width - w0;
                in.tables(a, c_base + w0, n);
                in.row(a, row, c_base + w0, n, false);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (i < n) { s += in.value(a, i); t += in.grad(a, i); }
            }
            unit_sum2<1024>(s, t, sh);
            mean = s * a.inv_width; dmean = t * a.inv_width;
            s = t = 0.0f;
        }
        for (int w0 = threadIdx.x * NV; w0 < a.width; w0 += 1024 * NV) {
            const int n = a.width - w0;
            in.tables(a, c_base + w0, n);
            in.row(a, row, c_base + w0, n, false);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float d = i < n ? in.value(a, i) - mean : 0.0f;
                s = fmaf(d, d, s);
                if (i < n) t = fmaf(in.grad(a, i), d, t);
            }
        }
        unit_sum2<1024>(s, t, sh);
        const float q = rsqrtf(fmaf(s, a.inv_width, a.eps)), proj = t * a.inv_width * q;
        if (a.part && threadIdx.x == 0) a.stats[unit] = make_float4(mean, q, dmean, proj);
        for (int w0 = threadIdx.x * NV; w0 < a.width; w0 += 1024 * NV) {
            const int c = c_base + w0, n = a.width - w0;
            const int64_t at = row * a.channels + c;
            in.tables(a, c, n);
            in.row(a, row, c, n, true);
            float dv[NV], dz[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float vn = (in.value(a, i) - mean) * q;
                dv[i] = (in.grad(a, i) - dmean - vn * proj) * q;
                if (GATE) {
                    const float z = in.z[i], sg = sigmoid_f(z), slope = sg * fmaf(z, 1.0f - sg, 1.0f);
                    dz[i] = (a.gate_first ? dv[i] * in.x[i] : in.dy[i] * fmaf(vn, in.w[i], in.t[i])) * slope;
                    if (a.gate_first) dv[i] *= z * sg;
                } else {
                    dv[i] += in.dr[i];
                }
            }
            if (GATE) {
                store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                store_vec<M, NV>(static_cast<M*>(a.dz) + at, dz, n);
            } else {
                if (a.dresidual) store_vec<RM, NV>(static_cast<RM*>(a.dresidual) + at, dv, n);
                if (a.dx) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) dv[i] *= in.t[i];
                    store_vec<M, NV>(static_cast<M*>(a.dx) + at, dv, n);
                }
            }
        }
    }
}

template <typename T, typename RT, bool GATE>
__global__ __launch_bounds__(256) void k_norm_columns(const Norm a) {
    const int g = blockIdx.y, w0 = (blockIdx.z * 256 + threadIdx.x) * NV, c = g * a.width + w0, n = a.width - w0;
    if (n <= 0) return;
    NormColumns<T, RT, GATE> in;
    in.tables(a, c, n);
    float sum[GATE ? 2 : 3][NV] = {};
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float4 st = a.stats[row * a.groups + g];           // mean, q, dmean, proj
        in.row(a, row, c, n, true);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float vn = (in.value(a, i) - st.x) * st.y;
            const float body = GATE && !a.gate_first ? in.dy[i] * in.gate(i) : in.dy[i];
            sum[0][i] = fmaf(body, vn, sum[0][i]);
            sum[1][i] += body;
            if (!GATE) {
                const float dv = fmaf(in.grad(a, i) - st.z - vn * st.w, st.y, in.dr[i]);
                sum[GATE ? 0 : 2][i] = fmaf(dv, in.x[i], sum[GATE ? 0 : 2][i]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < (GATE ? 2 : 3); ++j)
        if (a.want[j]) store_vec<float, NV>(a.part + ((int64_t)blockIdx.x * 3 + j) * a.channels + c, sum[j], n);
}

// 32 columns by 32 slices of the partial rows: 2048 of them, 1001 wide, in 7.3 us (64 columns by 16: 9.2 us; 16 by 64
// are slower for wide rows, 9.1 against 5.5 us at 1024 of 2048).
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_reduce(const float* __restrict__ part, int n_part, int channels, float* dweight,
                                                      float* dbias, float* dscale) {
    __shared__ float sh[16][32];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col, j = blockIdx.y;
    float* out = j == 0 ? dweight : j == 1 ? dbias : dscale;
    if (!out) return;
    float s = c < channels ? sum_strided(part + (int64_t)j * channels + c, slice, 32, n_part, 3 * (int64_t)channels) : 0.0f;
    s = halve32(s, s);
    if ((threadIdx.x & 63) < 32) sh[threadIdx.x >> 6][col] = s;
    __syncthreads();
    if (threadIdx.x < 32 && c < channels) {
        float t = 0.0f;
#pragma unroll
        for (int p = 0; p < 16; ++p) t += sh[p][col];
        out[c] = t;
    }
}

// ---- host --------------------------------------------------------------------------------------------
constexpr int NORM_MAX_WIDTH = 32768;

// Threads per row and steps of eight elements per thread: (16, 1) .. (1024, 4).  As few threads as hold the row in one
// step: their sums need fewer exchanges and no lanes idle (gradients of 30011 x 1000 in bfloat16 42 us with 128
// threads, 61 us with 256; of the gate 58 and 95 us).
template <int MOST, typename Fn>
int by_width_of_row(int width, Fn&& fn) {
    using std::integral_constant;
    if (width <= 128) return fn(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (width <= 256) return fn(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (width <= 512) return fn(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (width <= 1024) return fn(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    if (width <= 2048) return fn(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (width <= 4096) return fn(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (MOST <= 8192 || width <= 8192) return fn(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    if constexpr (MOST > 8192) {
        if (width <= 16384) return fn(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
        return fn(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
    }
}

// Rows up to this width stay in registers in the gradients too (4000 x 8192 bfloat16: 60 us, the gate 82 us, against 107 and
// 146 us by k_norm_bwd_wide); wider ones would spill (the gate at 1000 x 20000: 368 us, against 88 us).
constexpr int NORM_HELD = 8192;

// Blocks that walk over the rows in the backward pass, each with a row of partial sums: about four wavefronts for
// each of the 1024 SIMDs.
inline int norm_bwd_blocks(const mfcc_norm_args* a) {
    const int width = a->channels / a->groups, per = width <= 128 ? 16 : width <= 256 ? 8 : width <= 512 ? 4 : 1;
    const int64_t blocks = width <= 512 ? 1024 : width <= 1024 ? 2048 : width <= 4096 ? 1024 : 512;
    const int64_t tiles = width > NORM_HELD ? ceil_div(width, 256 * NV) : 1;
    const int64_t most = std::max<int64_t>(1, (width > NORM_HELD ? 2048 : blocks) / (a->groups * tiles));
    return (int)std::min<int64_t>(ceil_div(a->rows, per), most);
}
inline size_t norm_bwd_space(const mfcc_norm_args* a) {
    const size_t stats = a->channels / a->groups > NORM_HELD ? (size_t)a->rows * a->groups * sizeof(float4) : 0;
    return stats + (size_t)norm_bwd_blocks(a) * 3 * (size_t)a->channels * sizeof(float);
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
    f.room = has_room(f.x, f.x_stride, NV) && has_room(f.z, f.z_stride, NV) && has_room(f.residual, f.residual_stride, NV) &&
             has_room(f.r_in, f.r_stride, NV) && has_room(f.dy, f.dy_stride, NV) && has_room(f.dr, f.dr_stride, NV);
    return f;
}

template <typename T, typename RT, bool GATE>
int norm_forward(const mfcc_norm_args* a, hipStream_t st) {
    if (a->rows == 0) return MFCC_OK;
    const Norm f = norm_args(a);
    return by_width_of_row<NORM_MAX_WIDTH>(f.width, [&](auto tpu, auto it) {
        constexpr int TPU = decltype(tpu)::value, IT = decltype(it)::value, PER = norm_block(TPU) / TPU;
        const int64_t blocks = ceil_div(f.rows * f.groups, PER);
        if (blocks * norm_block(TPU) > 0xffffffffll) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
        hipLaunchKernelGGL((k_norm_fwd<T, RT, GATE, TPU, IT>), dim3((unsigned)blocks), dim3(norm_block(TPU)), 0, st, f);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

template <typename T, typename RT, bool GATE>
int norm_backward(const mfcc_norm_args* a, hipStream_t st) {
    Norm f = norm_args(a);
    if (!a->d_dscale && !GATE) f.x = nullptr;
    const int blocks = norm_bwd_blocks(a);
    f.want[0] = a->d_dweight; f.want[1] = a->d_dbias; f.want[2] = a->d_dscale;
    const bool sums = f.want[0] || f.want[1] || f.want[2];
    if (sums && ceil_div(f.channels, 32) > 0x3fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
    const bool wide = f.width > NORM_HELD;
    if (sums) {
        f.stats = static_cast<float4*>(a->d_workspace);
        f.part = static_cast<float*>(a->d_workspace) + (wide ? f.rows * f.groups * 4 : 0);
    }
    if (blocks > 0 && wide) {
        const unsigned tiles = (unsigned)ceil_div(f.width, 256 * NV);
        const int64_t units = std::min<int64_t>(f.rows * f.groups, 1 << 16);
        hipLaunchKernelGGL((k_norm_bwd_wide<T, RT, GATE>), dim3((unsigned)units), dim3(1024), 0, st, f);
        if (sums)
            hipLaunchKernelGGL((k_norm_columns<T, RT, GATE>), dim3((unsigned)blocks, (unsigned)f.groups, tiles), dim3(256), 0, st, f);
        PACKED_LAUNCHED();
    } else if (blocks > 0) {
        const int rc = by_width_of_row<NORM_HELD>(f.width, [&](auto tpu, auto it) {
            constexpr int TPU = decltype(tpu)::value, IT = decltype(it)::value;
            hipLaunchKernelGGL((k_norm_bwd<T, RT, GATE, TPU, IT>), dim3((unsigned)blocks, (unsigned)f.groups),
                               dim3(norm_block(TPU)), 0, st, f);
            PACKED_LAUNCHED();
            return (int)MFCC_OK;
        });
        if (rc) return rc;
    }
    if (sums) {
        hipLaunchKernelGGL(k_norm_reduce<T>, dim3((unsigned)ceil_div(f.channels, 32), 3), dim3(1024), 0, st, f.part, blocks,
                           f.channels, a->d_dweight, a->d_dbias, a->d_dscale);
        PACKED_LAUNCHED();
    }
    return (int)MFCC_OK;
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
