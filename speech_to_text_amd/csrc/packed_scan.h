// Selective state space scan over packed rows: forward, gradients, single tokens.
//   d = softplus(delta + bias);  h[n] = exp(d A[n]) h[n] + d u B[n];  y = sum_n C[n] h[n] + D u
//
// The recurrence is split over time into chunks.  For one chunk h_out = exp(A sum(d)) h_in + h_local, so
//   1. k_scan_sum    every chunk by itself from a zero state: h_local and sum(d)
//   2. k_scan_carry  the states between the chunks (a scan over chunks, one column per (n, channel))
//   3. k_scan_fwd    every chunk again, now from its true state, writing y.
// The gradient g of h runs the other way, g_t = C_t dy_t + a_{t+1} g_{t+1}, and is split the same way; its
// local part needs the running product of the a_t only, so pass 1 forms both with one exp per element.
// A chunk that holds the start of a sequence lets nothing through (its decay counts as zero).
//
// Bound by vector issue, not memory: per (row, channel, n) one exp (8 SIMD cycles per wavefront) and four to
// five plain operations (2.6 each) per pass against 6 / N bytes in 16-bit types.
#pragma once
#include "packed.h"

namespace packed {

constexpr float SCAN_LOG2E = LOG2E;
constexpr int SCAN_TILE = 32;       // rows of B and C staged in LDS at a time (forward kernels)

struct Scan {
    const void *u, *delta, *B, *C, *dy;
    int64_t u_stride, delta_stride, B_stride, C_stride, dy_stride, y_stride;
    const float *A, *D, *bias, *initial, *dfinal;
    const int64_t* off;
    void *y, *du, *ddelta;
    float *final, *dinitial;
    float *hst, *gst, *dsum;        // states entering each chunk from the left / right, sum of d: (chunk, n, channel), (chunk, channel)
    int32_t* reset;                 // chunk holds a sequence start
    float *part_bc, *part_A, *part_D, *part_bias;
    int64_t rows;
    int n_seqs, channels, state, groups, per, chunk, n_chunks, blocks_per_group, softplus, zero_rest;
};

template <typename M>
__device__ __forceinline__ float step_of(const Scan& a, M raw, float bias) {
    const float v = widen(raw) + bias;
    return a.softplus ? softplus_f(v) : v;
}

// Channels of one workgroup of the kernels with a lane per channel: whole wavefronts, spread evenly over as
// few workgroups of at most four wavefronts as a group of channels needs.
inline int scan_block(int per) {
    const int waves = (int)ceil_div(per, WAVE), blocks = (int)ceil_div(waves, 4);
    return WAVE * (int)ceil_div(waves, blocks);
}

// One row of B or C in LDS, read by all lanes at once.
template <int NP>
__device__ __forceinline__ void row_of(float (&v)[NP], const float* p) {
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p + n);
        v[n] = q.x; v[n + 1] = q.y; v[n + 2] = q.z; v[n + 3] = q.w;
    }
}

template <typename M, int NP>
__device__ __forceinline__ void stage_rows(float* lds, const M* __restrict__ src, int64_t stride, int64_t row, int count,
                                           int state) {
    for (int i = threadIdx.x; i < count * NP; i += blockDim.x) {
        const int n = i % NP;
        lds[i] = n < state ? widen(src[(row + i / NP) * stride + n]) : 0.0f;
    }
}

template <int NP>
__device__ __forceinline__ void load_rates(float (&A2)[NP], const Scan& a, int c) {
#pragma unroll
    for (int n = 0; n < NP; ++n) A2[n] = n < a.state ? a.A[(int64_t)c * a.state + n] * SCAN_LOG2E : 0.0f;
}

// Pass 1.  A lane holds a channel and all its states; B and C come from LDS.
template <typename T, int NP, bool BACK>
__global__ __launch_bounds__(256) void k_scan_sum(const Scan a) {
    using M = typename T::mem;
    __shared__ float sB[SCAN_TILE * NP], sC[BACK ? SCAN_TILE * NP : 1];
    const int n_blocks = a.groups * a.blocks_per_group;
    const int cb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int g = cb / a.blocks_per_group;
    const int in_group = (cb % a.blocks_per_group) * blockDim.x + threadIdx.x;
    const bool live = in_group < a.per;
    const int c = g * a.per + (live ? in_group : 0);
    const int64_t r0 = (int64_t)k * a.chunk, r1 = min(r0 + a.chunk, a.rows);
    const M* u = static_cast<const M*>(a.u) + c;
    const M* delta = static_cast<const M*>(a.delta) + c;
    const M* dy = static_cast<const M*>(a.dy) + c;
    const M* B = static_cast<const M*>(a.B) + (int64_t)g * a.state;
    const M* C = static_cast<const M*>(a.C) + (int64_t)g * a.state;
    const float bias = a.bias ? a.bias[c] : 0.0f;

    float A2[NP], h[NP], P[NP], R[NP];
    load_rates<NP>(A2, a, c);
#pragma unroll
    for (int n = 0; n < NP; ++n) { h[n] = 0.0f; P[n] = 1.0f; R[n] = 0.0f; }
    float sum = 0.0f;
    bool reset = false;            // a sequence start was passed: the reverse part is complete

    Place q = find_row(a.off, a.n_seqs, a.rows, r0);
    for (int64_t t0 = r0; t0 < r1; t0 += SCAN_TILE) {
        const int64_t t1 = min(t0 + SCAN_TILE, r1);
        __syncthreads();
        stage_rows<M, NP>(sB, B, a.B_stride, t0, (int)(t1 - t0), a.state);
        if (BACK) stage_rows<M, NP>(sC, C, a.C_stride, t0, (int)(t1 - t0), a.state);
        __syncthreads();
        for (int64_t r = t0; r < t1;) {
            if (r >= q.until) q = find_row(a.off, a.n_seqs, a.rows, r);
            const int64_t r2 = min(t1, q.until);
            if (!q.inside || r == q.start) {
                reset = true;
                sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    h[n] = q.inside && a.initial && n < a.state ? a.initial[((int64_t)q.s * a.channels + c) * a.state + n] : 0.0f;
            }
            if (!q.inside) { r = r2; continue; }
            for (; r < r2; ++r) {
                const float d = step_of(a, delta[r * a.delta_stride], bias);
                const float du = d * widen(u[r * a.u_stride]);
                float b[NP], cc[NP];
                row_of<NP>(b, sB + (r - t0) * NP);
                if (BACK && !reset) {
                    row_of<NP>(cc, sC + (r - t0) * NP);
                    const float dv = widen(dy[r * a.dy_stride]);
                    const bool last = a.dfinal && r + 1 == q.end;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const float e = exp2_hw(d * A2[n]);
                        float v = cc[n] * dv;
                        if (last && n < a.state) v += a.dfinal[((int64_t)q.s * a.channels + c) * a.state + n];
                        P[n] *= e;
                        R[n] = fmaf(P[n], v, R[n]);
                        h[n] = fmaf(e, h[n], du * b[n]);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NP; ++n) h[n] = fmaf(exp2_hw(d * A2[n]), h[n], du * b[n]);
                }
                sum += d;
            }
        }
    }
    if (!live) return;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < a.state) {
            const int64_t at = ((int64_t)k * a.state + n) * a.channels + c;
            a.hst[at] = h[n];
            if (BACK) a.gst[at] = R[n];
        }
    a.dsum[(int64_t)k * a.channels + c] = sum;
    if (c == 0) a.reset[k] = reset;
}

// Pass 2, in place: hst[k] (and, from the right, gst[k]) becomes the state that enters chunk k.  64 columns
// by 16 segments of the chunks: each segment's own composition, then the ones before it, then the segment.
template <typename T>
__global__ __launch_bounds__(1024) void k_scan_carry(const Scan a) {
    __shared__ float sD[16][64], sH[16][64];
    const int lane = threadIdx.x & 63, seg = threadIdx.x >> 6;
    const bool right = blockIdx.y == 1;
    float* st = right ? a.gst : a.hst;
    const int64_t m = (int64_t)a.state * a.channels;
    const int64_t e = (int64_t)blockIdx.x * 64 + lane;
    const bool live = e < m;
    const int n = live ? (int)(e / a.channels) : 0, c = live ? (int)(e % a.channels) : 0;
    const float A2 = a.A[(int64_t)c * a.state + n] * SCAN_LOG2E;
    const int len = (a.n_chunks + 15) / 16;
    const int k0 = min(seg * len, a.n_chunks), k1 = min(k0 + len, a.n_chunks);
    float D = 1.0f, H = 0.0f;
    if (live)
        for (int i = k0; i < k1; ++i) {
            const int k = right ? a.n_chunks - 1 - i : i;
            const float v = st[k * m + e];
            const bool cut = a.reset[k] != 0;
            const float dec = exp2_hw(A2 * a.dsum[(int64_t)k * a.channels + c]);
            H = cut ? v : fmaf(dec, H, v);
            D = cut ? 0.0f : D * dec;
        }
    sD[seg][lane] = D; sH[seg][lane] = H;
    __syncthreads();
    if (!live) return;
    float carry = 0.0f;
    // D == 0 also where a chunk of the segment is cut: nothing passes, whatever the carry is
    for (int s = 0; s < seg; ++s) carry = sD[s][lane] == 0.0f ? sH[s][lane] : fmaf(sD[s][lane], carry, sH[s][lane]);
    for (int i = k0; i < k1; ++i) {
        const int k = right ? a.n_chunks - 1 - i : i;
        const float v = st[k * m + e];
        const bool cut = a.reset[k] != 0;
        const float dec = exp2_hw(A2 * a.dsum[(int64_t)k * a.channels + c]);
        st[k * m + e] = carry;
        carry = cut ? v : fmaf(dec, carry, v);
    }
}

// Pass 3: y, and the states that sequences leave behind.
template <typename T, int NP>
__global__ __launch_bounds__(256) void k_scan_fwd(const Scan a) {
    using M = typename T::mem;
    __shared__ float sB[SCAN_TILE * NP], sC[SCAN_TILE * NP];
    const int n_blocks = a.groups * a.blocks_per_group;
    const int cb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int g = cb / a.blocks_per_group;
    const int in_group = (cb % a.blocks_per_group) * blockDim.x + threadIdx.x;
    const bool live = in_group < a.per;
    const int c = g * a.per + (live ? in_group : 0);
    const int64_t r0 = (int64_t)k * a.chunk, r1 = min(r0 + a.chunk, a.rows);
    const M* u = static_cast<const M*>(a.u) + c;
    const M* delta = static_cast<const M*>(a.delta) + c;
    M* y = static_cast<M*>(a.y) + c;
    const M* B = static_cast<const M*>(a.B) + (int64_t)g * a.state;
    const M* C = static_cast<const M*>(a.C) + (int64_t)g * a.state;
    const float bias = a.bias ? a.bias[c] : 0.0f;
    const float skip = a.D ? a.D[c] : 0.0f;

    float A2[NP], h[NP];
    load_rates<NP>(A2, a, c);
#pragma unroll
    for (int n = 0; n < NP; ++n)
        h[n] = a.n_chunks > 1 && n < a.state ? a.hst[((int64_t)k * a.state + n) * a.channels + c] : 0.0f;

    Place q = find_row(a.off, a.n_seqs, a.rows, r0);
    for (int64_t t0 = r0; t0 < r1; t0 += SCAN_TILE) {
        const int64_t t1 = min(t0 + SCAN_TILE, r1);
        __syncthreads();
        stage_rows<M, NP>(sB, B, a.B_stride, t0, (int)(t1 - t0), a.state);
        stage_rows<M, NP>(sC, C, a.C_stride, t0, (int)(t1 - t0), a.state);
        __syncthreads();
        for (int64_t r = t0; r < t1;) {
            if (r >= q.until) q = find_row(a.off, a.n_seqs, a.rows, r);
            const int64_t r2 = min(t1, q.until);
            if (!q.inside) {
                if (a.zero_rest && live)
                    for (; r < r2; ++r) y[r * a.y_stride] = narrow<M>(0.0f);
                r = r2;
                continue;
            }
            if (r == q.start) {
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    h[n] = a.initial && n < a.state ? a.initial[((int64_t)q.s * a.channels + c) * a.state + n] : 0.0f;
            }
            for (; r < r2; ++r) {
                const float uv = widen(u[r * a.u_stride]);
                const float d = step_of(a, delta[r * a.delta_stride], bias);
                const float du = d * uv;
                float b[NP], cc[NP];
                row_of<NP>(b, sB + (r - t0) * NP);
                row_of<NP>(cc, sC + (r - t0) * NP);
                float acc = skip * uv;
                if (!a.D) acc = 0.0f;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    h[n] = fmaf(exp2_hw(d * A2[n]), h[n], du * b[n]);
                    acc = fmaf(cc[n], h[n], acc);
                }
                if (live) y[r * a.y_stride] = narrow<M>(acc);
            }
            if (a.final && r == q.end && live) {
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    if (n < a.state) a.final[((int64_t)q.s * a.channels + c) * a.state + n] = h[n];
            }
        }
    }
}

// Sequences without rows (and those whose offsets do not lie within the rows): the state passes through,
// and so does its gradient.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_empty(const int64_t* __restrict__ off, int64_t rows, int64_t size,
                                                    const float* __restrict__ from, float* __restrict__ to) {
    const int64_t s = blockIdx.x;
    const int64_t start = off ? off[s] : 0, end = off ? min(off[s + 1], rows) : rows;
    if (start >= 0 && start < end) return;
    for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.y * 256)
        to[s * size + i] = from ? from[s * size + i] : 0.0f;
}

// ---- gradients ---------------------------------------------------------------------------------------
// A lane holds four of a channel's states (LPC = NP / 4 lanes per channel), a workgroup of four wavefronts
// 4 * 64 / LPC channels of one group and one chunk of rows.  The chunk's d, u, dy, B and C lie in LDS.  The
// chunk is swept once forward, keeping the state at every eighth row, and then eight rows at a time from
// its end: forward again with all eight states and decays in registers, and back over them.
//   g = C dy + G;  dC = dy h;  dB = d u g;  G = a g;  w = G h_before;  dA += d w;
//   du = d sum(g B) + D dy;  dd = u sum(g B) + sum(A w)
// Sums over n stay in the LPC lanes of a channel; dB and dC are summed over the channels of the wavefront
// (v_permlane swaps halve eight values to two, then rotations within a row of lanes), over the four
// wavefronts in LDS, and over the workgroups of a group by k_scan_reduce: a fixed order throughout.
constexpr int SUB = 8;

template <int NP> constexpr int bwd_lpc() { return NP / 4; }
template <int NP> constexpr int bwd_channels() { return 4 * WAVE / bwd_lpc<NP>(); }
template <int NP> constexpr int bwd_rows() { return bwd_channels<NP>() >= 256 ? 16 : bwd_channels<NP>() >= 128 ? 32 : 64; }

template <int LPC>
__device__ __forceinline__ float sum_states(float v) {       // over the LPC neighbouring lanes of a channel
    if (LPC >= 2) v += dpp<0xB1>(v);                          // quad_perm [1, 0, 3, 2]
    if (LPC >= 4) v += dpp<0x4E>(v);                          // quad_perm [2, 3, 0, 1]
    if (LPC >= 8) v += dpp<0x141>(v);                         // row_half_mirror
    if (LPC >= 16) v += dpp<0x140>(v);                        // row_mirror
    return v;
}

template <int LPC>
__device__ __forceinline__ float sum_channels(float v) {     // over the lanes of a row of 16 with equal lane % LPC
    if (LPC <= 1) v += dpp<0x121>(v);                         // row_ror:1, 2, 4, 8
    if (LPC <= 2) v += dpp<0x122>(v);
    if (LPC <= 4) v += dpp<0x124>(v);
    if (LPC <= 8) v += dpp<0x128>(v);
    return v;
}

template <typename T, int NP>
__global__ __launch_bounds__(256) void k_scan_bwd(const Scan a) {
    using M = typename T::mem;
    constexpr int LPC = bwd_lpc<NP>(), CPW = WAVE / LPC, CPB = 4 * CPW, MAXR = bwd_rows<NP>(), NSUB = MAXR / SUB;
    __shared__ float sd[MAXR * CPB];                 // d, later the gradient of d
    __shared__ M su[MAXR * CPB];                     // u, later its gradient
    __shared__ M sdy[MAXR * CPB];
    __shared__ float sB[MAXR * NP], sC[MAXR * NP];
    __shared__ float slab[4][SUB][2][NP];
    __shared__ int sseq[MAXR], sflag[MAXR];
    __shared__ float ssum[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_blocks = a.groups * a.blocks_per_group;
    const int cb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int g = cb / a.blocks_per_group, gb = cb % a.blocks_per_group;
    const int64_t r0 = (int64_t)k * a.chunk;
    const int len = (int)min((int64_t)a.chunk, a.rows - r0);
    const int c_base = g * a.per + gb * CPB, n_ch = min(a.per - gb * CPB, CPB);
    enum { OUT = 4, START = 1, END = 2 };

    if (tid < len) {
        const Place q = find_row(a.off, a.n_seqs, a.rows, r0 + tid);
        sseq[tid] = q.s;
        sflag[tid] = !q.inside ? (OUT | START | END)
                               : (r0 + tid == q.start ? START : 0) | (r0 + tid + 1 == q.end ? END : 0);
    }
    __syncthreads();
    {   // rows outside every sequence count as zero, whatever they hold
        const int ch = tid % CPB;
        const float bias = a.bias && ch < n_ch ? a.bias[c_base + ch] : 0.0f;
        float dD = 0.0f;
        for (int t = tid / CPB; t < len; t += 256 / CPB) {
            float d = 0.0f; M uv = (M)0.0f, dv = (M)0.0f;
            if (ch < n_ch && !(sflag[t] & OUT)) {
                const int64_t row = r0 + t;
                d = step_of(a, static_cast<const M*>(a.delta)[row * a.delta_stride + c_base + ch], bias);
                uv = static_cast<const M*>(a.u)[row * a.u_stride + c_base + ch];
                dv = static_cast<const M*>(a.dy)[row * a.dy_stride + c_base + ch];
                dD = fmaf(widen(uv), widen(dv), dD);
            }
            sd[t * CPB + ch] = d; su[t * CPB + ch] = uv; sdy[t * CPB + ch] = dv;
        }
        ssum[tid] = dD;
        for (int i = tid; i < len * NP; i += 256) {
            const int t = i / NP, n = i % NP;
            const bool in = n < a.state && !(sflag[t] & OUT);
            sB[i] = in ? widen(static_cast<const M*>(a.B)[(r0 + t) * a.B_stride + (int64_t)g * a.state + n]) : 0.0f;
            sC[i] = in ? widen(static_cast<const M*>(a.C)[(r0 + t) * a.C_stride + (int64_t)g * a.state + n]) : 0.0f;
        }
        __syncthreads();
        if (a.part_D && tid < n_ch) {
            float s = 0.0f;
            for (int i = tid; i < 256; i += CPB) s += ssum[i];
            a.part_D[(int64_t)k * a.channels + c_base + tid] = s;
        }
    }

    const int nq = lane % LPC, chl = wave * CPW + lane / LPC;       // the lane's states and channel
    const bool live = chl < n_ch;
    const int c = c_base + (live ? chl : 0), n0 = nq * 4;
    const float skip = a.D ? a.D[c] : 0.0f;
    float A[4], A2[4], h[4], G[4], dA[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        A[i] = n0 + i < a.state ? a.A[(int64_t)c * a.state + n0 + i] : 0.0f;
        A2[i] = A[i] * SCAN_LOG2E;
        const bool has = a.n_chunks > 1 && live && n0 + i < a.state;
        const int64_t at = ((int64_t)k * a.state + n0 + i) * a.channels + c;
        h[i] = has ? a.hst[at] : 0.0f;
        G[i] = has ? a.gst[at] : 0.0f;
        dA[i] = 0.0f;
    }
    auto enter = [&](float (&v)[4], int t, const float* from) {       // a state of the sequence of row t
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = from && live && !(sflag[t] & OUT) && n0 + i < a.state
                       ? from[((int64_t)sseq[t] * a.channels + c) * a.state + n0 + i] : 0.0f;
    };
    auto four = [&](const float* p) { return *reinterpret_cast<const float4*>(p); };

    const int n_sub = (len + SUB - 1) / SUB;
    float keep[NSUB][4];
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[s][i] = h[i];
        if (s + 1 < n_sub) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const int t = s * SUB + j;
                if (__builtin_amdgcn_readfirstlane(sflag[t]) & START) enter(h, t, a.initial);
                const float d = sd[t * CPB + chl], du = d * widen(su[t * CPB + chl]);
                const float4 b = four(sB + t * NP + n0);
                h[0] = fmaf(exp2_hw(d * A2[0]), h[0], du * b.x);
                h[1] = fmaf(exp2_hw(d * A2[1]), h[1], du * b.y);
                h[2] = fmaf(exp2_hw(d * A2[2]), h[2], du * b.z);
                h[3] = fmaf(exp2_hw(d * A2[3]), h[3], du * b.w);
            }
        }
    }
#pragma unroll
    for (int s = NSUB - 1; s >= 0; --s) {
        if (s >= n_sub) continue;
        float hs[SUB + 1][4], ea[SUB][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) hs[0][i] = keep[s][i];
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int t = s * SUB + j;
            if (t < len) {
                float prev[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) prev[i] = hs[j][i];
                if (__builtin_amdgcn_readfirstlane(sflag[t]) & START) enter(prev, t, a.initial);
                const float d = sd[t * CPB + chl], du = d * widen(su[t * CPB + chl]);
                const float4 b4 = four(sB + t * NP + n0);
                const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ea[j][i] = exp2_hw(d * A2[i]);
                    hs[j + 1][i] = fmaf(ea[j][i], prev[i], du * b[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) { ea[j][i] = 1.0f; hs[j + 1][i] = 0.0f; }
            }
        }
#pragma unroll
        for (int j = SUB - 1; j >= 0; --j) {
            const int t = s * SUB + j;
            float red[8];
            if (t < len) {
                const int flag = __builtin_amdgcn_readfirstlane(sflag[t]);
                float prev[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) prev[i] = hs[j][i];
                if (flag & START) enter(prev, t, a.initial);
                if (flag & END) enter(G, t, a.dfinal);
                const float d = sd[t * CPB + chl], uv = widen(su[t * CPB + chl]), dv = widen(sdy[t * CPB + chl]);
                const float du = d * uv;
                const float4 b4 = four(sB + t * NP + n0), c4 = four(sC + t * NP + n0);
                const float b[4] = {b4.x, b4.y, b4.z, b4.w}, cc[4] = {c4.x, c4.y, c4.z, c4.w};
                float gB = 0.0f, wA = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float gr = fmaf(cc[i], dv, G[i]);
                    red[i] = du * gr;
                    red[4 + i] = dv * hs[j + 1][i];
                    gB = fmaf(gr, b[i], gB);
                    G[i] = ea[j][i] * gr;
                    const float w = G[i] * prev[i];
                    dA[i] = fmaf(d, w, dA[i]);
                    wA = fmaf(A[i], w, wA);
                }
                if ((flag & START) && a.dinitial && !(flag & OUT) && live) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n0 + i < a.state) a.dinitial[((int64_t)sseq[t] * a.channels + c) * a.state + n0 + i] = G[i];
                }
                gB = sum_states<LPC>(gB);
                wA = sum_states<LPC>(wA);
                if (nq == 0) {
                    sd[t * CPB + chl] = fmaf(uv, gB, wA);
                    su[t * CPB + chl] = narrow<M>(fmaf(d, gB, skip * dv));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) red[i] = 0.0f;
            }
            const float w0 = halve32(red[0], red[4]), w1 = halve32(red[1], red[5]);
            const float w2 = halve32(red[2], red[6]), w3 = halve32(red[3], red[7]);
            const float v0 = sum_channels<LPC>(halve16(w0, w2)), v1 = sum_channels<LPC>(halve16(w1, w3));
            if ((lane & 15) < LPC) {
                float* p = &slab[wave][j][lane >> 5][(lane & 15) * 4 + ((lane >> 4) & 1) * 2];
                p[0] = v0; p[1] = v1;
            }
        }
        __syncthreads();
        for (int i = tid; i < SUB * 2 * NP; i += 256) {
            const int j = i / (2 * NP), w = i / NP & 1, n = i % NP, t = s * SUB + j;
            if (t < len)
                a.part_bc[(((int64_t)w * a.blocks_per_group + gb) * a.rows + r0 + t) * a.groups * NP + (int64_t)g * NP + n] =
                    (slab[0][j][w][n] + slab[1][j][w][n]) + (slab[2][j][w][n] + slab[3][j][w][n]);
        }
        __syncthreads();
    }
    if (live) {
        float* p = a.part_A + ((int64_t)k * a.channels + c) * NP + n0;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = dA[i];
    }
    __syncthreads();
    const int ch = tid % CPB;
    float db = 0.0f;
    if (ch < n_ch) {
        const float bias = a.bias ? a.bias[c_base + ch] : 0.0f;
        for (int t = tid / CPB; t < len; t += 256 / CPB) {
            const int64_t at = (r0 + t) * a.channels + c_base + ch;
            float v = sd[t * CPB + ch];
            if (sflag[t] & OUT) v = 0.0f;
            else if (a.softplus) v *= sigmoid_f(widen(static_cast<const M*>(a.delta)[(r0 + t) * a.delta_stride + c_base + ch]) + bias);
            db += v;
            static_cast<M*>(a.ddelta)[at] = narrow<M>(v);
            static_cast<M*>(a.du)[at] = su[t * CPB + ch];
        }
    }
    ssum[tid] = db;
    __syncthreads();
    if (a.part_bias && tid < n_ch) {
        float s = 0.0f;
        for (int i = tid; i < 256; i += CPB) s += ssum[i];
        a.part_bias[(int64_t)k * a.channels + c_base + tid] = s;
    }
}

// out[e] = sum over parts of part[p][e]; rows of `padded` columns of which the first `inner` are kept.
template <typename M, typename T>
__global__ __launch_bounds__(256) void k_scan_reduce(const float* __restrict__ part, int64_t n_part, int64_t m, int padded,
                                                     int inner, M* __restrict__ out) {
    __shared__ float sh[4][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < m; e0 += (int64_t)gridDim.x * 64) {
        const int64_t e = e0 + lane;
        float s = 0.0f;
        if (e < m)
            for (int64_t p = slice; p < n_part; p += 4) s += part[p * m + e];
        sh[slice][lane] = s;
        __syncthreads();
        if (slice == 0 && e < m && e % padded < inner)
            out[e / padded * inner + e % padded] = narrow<M>((sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]));
        __syncthreads();
    }
}

// ---- single tokens --------------------------------------------------------------------------------------
// Bound by the state: 8 N bytes per channel read and written.  Four states per lane, 16-byte accesses.
struct ScanStep {
    const void *u, *delta, *B, *C;
    int64_t u_stride, delta_stride, B_stride, C_stride, y_stride;
    const float *A, *D, *bias, *state_in;
    float* state_out;
    const int32_t* slots;
    void* y;
    int batch, n_slots, channels, state, per, softplus;
};

// Entries that name the same slot are successive tokens of that sequence and are taken by the first of
// them; a slot outside the pool gives a zero row and touches no state.
template <typename T, int NP>
__global__ __launch_bounds__(256) void k_scan_step(const ScanStep a) {
    using M = typename T::mem;
    constexpr int LPC = NP / 4;
    const int e0 = blockIdx.y;
    int slot = e0;
    bool again = false;
    if (a.slots) {
        slot = a.slots[e0];
        const SlotUse use = slot_use(a.slots, a.batch, e0);
        if (use.before && (unsigned)slot < (unsigned)a.n_slots) return;
        again = use.after;
    }
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int nq = (int)(id % LPC), n0 = nq * 4;
    const bool live = id / LPC < a.channels;
    const int c = live ? (int)(id / LPC) : 0;
    M* y = static_cast<M*>(a.y) + c;
    if ((unsigned)slot >= (unsigned)a.n_slots) {
        if (live && nq == 0) y[(int64_t)e0 * a.y_stride] = narrow<M>(0.0f);
        return;
    }
    const int left = live ? max(a.state - n0, 0) : 0;           // of the lane's four states, how many exist
    const int64_t at = ((int64_t)slot * a.channels + c) * a.state + n0;
    const int64_t bc = (int64_t)(c / a.per) * a.state + n0;
    float h[4], A2[4];
    load_vec<float, 4>(h, a.state_in + at, left);
    load_vec<float, 4>(A2, a.A + (int64_t)c * a.state + n0, left);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] *= SCAN_LOG2E;
    const float bias = a.bias ? a.bias[c] : 0.0f, skip = a.D ? a.D[c] : 0.0f;
    for (int e = e0; e < a.batch; ++e) {
        if (e != e0) {
            if (!again) break;
            if (a.slots[e] != slot) continue;
        }
        const float uv = widen(static_cast<const M*>(a.u)[(int64_t)e * a.u_stride + c]);
        float d = widen(static_cast<const M*>(a.delta)[(int64_t)e * a.delta_stride + c]) + bias;
        if (a.softplus) d = softplus_f(d);
        float b[4], cc[4];
        load_vec<M, 4>(b, static_cast<const M*>(a.B) + (int64_t)e * a.B_stride + bc, left);
        load_vec<M, 4>(cc, static_cast<const M*>(a.C) + (int64_t)e * a.C_stride + bc, left);
        float acc = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = fmaf(exp2_hw(d * A2[i]), h[i], d * uv * b[i]);
            acc = fmaf(cc[i], h[i], acc);
        }
        acc = sum_states<LPC>(acc);
        if (a.D) acc = fmaf(skip, uv, acc);
        if (live && nq == 0) y[(int64_t)e * a.y_stride] = narrow<M>(acc);
    }
    if (left > 0) store_vec<float, 4>(a.state_out + at, h, left);
}

// ---- host ------------------------------------------------------------------------------------------------
template <typename Fn>
int by_state(int state, Fn&& fn) {          // states padded to a power of two, four at least
    if (state <= 4) return fn(std::integral_constant<int, 4>{});
    if (state <= 8) return fn(std::integral_constant<int, 8>{});
    if (state <= 16) return fn(std::integral_constant<int, 16>{});
    if (state <= 32) return fn(std::integral_constant<int, 32>{});
    return fn(std::integral_constant<int, 64>{});
}
inline int padded_state(int state) {
    int np = 4;
    while (np < state) np *= 2;
    return np;
}

// Rows per chunk of the forward pass.  A chunk costs 16 bytes per state of traffic between the passes, so
// long ones are preferred while they leave about four wavefronts for every SIMD (256 CUs x 4); up to 64
// rows one pass without chunks is faster than three launches.
inline int scan_fwd_chunk(const mfcc_scan_args* a) {
    if (a->rows <= 64) return 64;
    const int64_t waves = (int64_t)a->groups * ceil_div(a->channels / a->groups, WAVE);
    for (int chunk : {256, 128, 64})
        if (waves * ceil_div(a->rows, chunk) >= 4 * 1024) return chunk;
    return 32;
}

inline int bwd_channels_of(int np) { return 4 * WAVE / (np / 4); }
inline int scan_bwd_chunk(const mfcc_scan_args* a) {
    const int cpb = bwd_channels_of(padded_state(a->state)), most = cpb >= 256 ? 16 : cpb >= 128 ? 32 : 64;
    const int64_t blocks = (int64_t)a->groups * ceil_div(a->channels / a->groups, cpb);
    int chunk = most;
    while (chunk > 16 && blocks * ceil_div(a->rows, chunk) < 1024) chunk /= 2;
    return chunk;
}

inline size_t round256(size_t v) { return (v + 255) / 256 * 256; }

struct ScanSpace {      // byte offsets into the workspace
    size_t hst = 0, gst = 0, dsum = 0, reset = 0, bc = 0, A = 0, D = 0, bias = 0, total = 0;
};
inline ScanSpace scan_space(const mfcc_scan_args* a, bool back) {
    ScanSpace s;
    const int chunk = back ? scan_bwd_chunk(a) : scan_fwd_chunk(a);
    const size_t nc = (size_t)ceil_div(a->rows, chunk), ch = (size_t)a->channels, np = (size_t)padded_state(a->state);
    size_t at = 0;
    auto take = [&](size_t floats) { const size_t o = at; at += round256(floats * 4); return o; };
    if (nc > 1) {
        s.hst = take(nc * a->state * ch);
        if (back) s.gst = take(nc * a->state * ch);
        s.dsum = take(nc * ch);
        s.reset = take(nc);
    }
    if (back) {
        const size_t bpg = (size_t)ceil_div(a->channels / a->groups, bwd_channels_of((int)np));
        s.bc = take(2 * bpg * (size_t)a->rows * a->groups * np);
        s.A = take(nc * ch * np);
        s.D = take(nc * ch);
        s.bias = take(nc * ch);
    }
    s.total = at;
    return s;
}

inline Scan scan_args(const mfcc_scan_args* a, bool back) {
    Scan f = {};
    f.u = a->d_u; f.delta = a->d_delta; f.B = a->d_B; f.C = a->d_C; f.dy = a->d_dy;
    f.u_stride = a->u_stride; f.delta_stride = a->delta_stride; f.B_stride = a->B_stride; f.C_stride = a->C_stride;
    f.dy_stride = a->dy_stride; f.y_stride = a->y_stride;
    f.A = a->d_A; f.D = a->d_D; f.bias = a->d_delta_bias; f.initial = a->d_initial; f.dfinal = a->d_dfinal;
    f.off = a->d_offsets; f.y = a->d_y; f.du = a->d_du; f.ddelta = a->d_ddelta; f.final = a->d_final;
    f.dinitial = a->d_dinitial;
    f.rows = a->rows; f.n_seqs = a->n_seqs; f.channels = a->channels; f.state = a->state; f.groups = a->groups;
    f.per = a->channels / a->groups; f.chunk = back ? scan_bwd_chunk(a) : scan_fwd_chunk(a);
    f.n_chunks = (int)ceil_div(a->rows, f.chunk);
    f.softplus = a->softplus; f.zero_rest = a->zero_rest;
    const ScanSpace s = scan_space(a, back);
    char* ws = static_cast<char*>(a->d_workspace);
    auto at = [&](size_t o) { return reinterpret_cast<float*>(ws + o); };
    f.hst = at(s.hst); f.gst = at(s.gst); f.dsum = at(s.dsum); f.reset = reinterpret_cast<int32_t*>(at(s.reset));
    f.part_bc = at(s.bc); f.part_A = at(s.A);
    f.part_D = a->d_dD ? at(s.D) : nullptr; f.part_bias = a->d_ddelta_bias ? at(s.bias) : nullptr;
    return f;
}

template <typename T>
int scan_empties(const mfcc_scan_args* a, const float* from, float* to, hipStream_t st) {
    if (!to || a->n_seqs == 0 || (!a->d_offsets && a->rows > 0)) return MFCC_OK;
    const int64_t size = (int64_t)a->channels * a->state;
    hipLaunchKernelGGL(k_scan_empty<T>, dim3((unsigned)a->n_seqs, (unsigned)std::min<int64_t>(ceil_div(size, 256), 64)), dim3(256),
                       0, st, a->d_offsets, a->rows, size, from, to);
    PACKED_LAUNCHED();
    return MFCC_OK;
}

template <typename T>
int scan_forward(const mfcc_scan_args* a, hipStream_t st) {
    Scan f = scan_args(a, false);
    const int block = scan_block(f.per);
    f.blocks_per_group = (int)ceil_div(f.per, block);
    const int64_t grid = (int64_t)f.groups * f.blocks_per_group * f.n_chunks;
    if (grid > 0x7fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
    if (a->rows > 0) {
        const int rc = by_state(a->state, [&](auto np) {
            constexpr int NP = decltype(np)::value;
            if (f.n_chunks > 1) {
                hipLaunchKernelGGL((k_scan_sum<T, NP, false>), dim3((unsigned)grid), dim3(block), 0, st, f);
                hipLaunchKernelGGL(k_scan_carry<T>, dim3((unsigned)ceil_div((int64_t)f.state * f.channels, 64), 1), dim3(1024),
                                   0, st, f);
            }
            hipLaunchKernelGGL((k_scan_fwd<T, NP>), dim3((unsigned)grid), dim3(block), 0, st, f);
            PACKED_LAUNCHED();
            return (int)MFCC_OK;
        });
        if (rc) return rc;
    }
    return scan_empties<T>(a, a->d_initial, a->d_final, st);
}

template <typename T>
int scan_backward(const mfcc_scan_args* a, hipStream_t st) {
    using M = typename T::mem;
    Scan f = scan_args(a, true);
    return by_state(a->state, [&](auto np) {
        constexpr int NP = decltype(np)::value;
        if (a->rows > 0) {
            const int block = scan_block(f.per);
            f.blocks_per_group = (int)ceil_div(f.per, block);
            const int64_t grid = (int64_t)f.groups * f.blocks_per_group * f.n_chunks;
            if (f.n_chunks > 1) {
                if (grid > 0x7fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
                hipLaunchKernelGGL((k_scan_sum<T, NP, true>), dim3((unsigned)grid), dim3(block), 0, st, f);
                hipLaunchKernelGGL(k_scan_carry<T>, dim3((unsigned)ceil_div((int64_t)f.state * f.channels, 64), 2), dim3(1024),
                                   0, st, f);
            }
            f.blocks_per_group = (int)ceil_div(f.per, bwd_channels<NP>());
            const int64_t grid2 = (int64_t)f.groups * f.blocks_per_group * f.n_chunks;
            if (grid2 > 0x7fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
            hipLaunchKernelGGL((k_scan_bwd<T, NP>), dim3((unsigned)grid2), dim3(256), 0, st, f);
            PACKED_LAUNCHED();
        }
        const int64_t m = a->rows * f.groups * NP;
        auto reduce = [&](const float* part, int64_t n_part, int64_t size, int padded, int inner, auto* out) {
            using O = std::remove_pointer_t<decltype(out)>;
            if (size == 0) return;
            const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(size, 64), 1 << 20);
            hipLaunchKernelGGL((k_scan_reduce<O, T>), dim3(blocks), dim3(256), 0, st, part, n_part, size, padded, inner, out);
        };
        reduce(f.part_bc, f.blocks_per_group, m, NP, f.state, static_cast<M*>(a->d_dB));
        reduce(f.part_bc + f.blocks_per_group * m, f.blocks_per_group, m, NP, f.state, static_cast<M*>(a->d_dC));
        reduce(f.part_A, f.n_chunks, (int64_t)f.channels * NP, NP, f.state, a->d_dA);
        if (a->d_dD) reduce(f.part_D, f.n_chunks, f.channels, 1, 1, a->d_dD);
        if (a->d_ddelta_bias) reduce(f.part_bias, f.n_chunks, f.channels, 1, 1, a->d_ddelta_bias);
        PACKED_LAUNCHED();
        return scan_empties<T>(a, a->d_dfinal, a->d_dinitial, st);
    });
}

template <typename T>
int scan_step(const mfcc_scan_args* a, int n_slots, const int32_t* slots, hipStream_t st) {
    ScanStep f = {};
    f.u = a->d_u; f.delta = a->d_delta; f.B = a->d_B; f.C = a->d_C;
    f.u_stride = a->u_stride; f.delta_stride = a->delta_stride; f.B_stride = a->B_stride; f.C_stride = a->C_stride;
    f.y_stride = a->y_stride; f.A = a->d_A; f.D = a->d_D; f.bias = a->d_delta_bias; f.state_in = a->d_initial;
    f.state_out = a->d_final; f.slots = slots; f.y = a->d_y; f.batch = (int)a->rows; f.n_slots = n_slots;
    f.channels = a->channels; f.state = a->state; f.per = a->channels / a->groups; f.softplus = a->softplus;
    return by_state(a->state, [&](auto np) {
        constexpr int NP = decltype(np)::value;
        hipLaunchKernelGGL((k_scan_step<T, NP>), dim3((unsigned)ceil_div((int64_t)a->channels * (NP / 4), 256), (unsigned)f.batch),
                           dim3(256), 0, st, f);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

}  // namespace packed
