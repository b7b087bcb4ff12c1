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
// Bound by vector issue, not memory: per (row, channel, n) one exp and three plain operations in the first sweep, four in
// the last one, against 6 / N bytes in 16-bit types.  A SIMD has one issue slot in four cycles.  An exp takes two; a plain
// operation takes one, or half where it is issued in a pair with one of another wavefront (2.6 cycles in a loop of
// nothing else).  16384 x 2048, 16 states, bfloat16: 118 + 11 + 150 us for the three passes.  By the counters the first
// sweep issues 50 M instructions (9.5 M of them exp and log), a third of them in pairs, in 51 M slots: 81 % of the slots of
// busy CUs, and CUs are busy 90 % of the time.  The last one issues 63 M, 36 % in pairs, in 61 M slots, 78 %.  With pairs
// throughout both would take two thirds of their time; a third of the instructions is softplus, staging and the loop.
// The first sweep is what the split costs: undivided, 2048 channels are 32 wavefronts for 1024 SIMDs.
#pragma once
#include "packed.h"

namespace packed {

constexpr int SCAN_TILE = 32;       // rows of B and C staged in LDS at a time (forward kernels)
constexpr int ZERO_ROW = SCAN_TILE;  // behind them one of zeros, for the missing rows of a group of four: with a step
                                     // of zero as well they change nothing, also behind an infinite row

// A log2(e), so that a decay is exp2(d rate): d A is rounded twice where exp(d A) would round it once, and a decay over
// rows with sum |d A| = X is off by up to X 2^-23 of itself.  For A <= 0 that is at most 2^-23 / e of the state (X exp(-X)
// <= 1 / e).  A second float of the product would cost two more operations per element, to four or five.  Also, a step of
// zero (a missing row too) decays by one whatever the rate: beyond the range of float32 it is the lowest number.
__device__ __forceinline__ float rate_of(float A) { return __builtin_elementwise_maximum(A * LOG2E, -3.40282347e38f); }   // a NaN stays

// Holds the LDS reads of the next row back until half of this row's states are done: hoisted by the compiler,
// the B and C of four rows take the registers of two wavefronts.
__device__ __forceinline__ void after(int& offset, float& state) { asm volatile("" : "+v"(offset), "+v"(state)); }

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

// d of a row.
template <typename M>
__device__ __forceinline__ float step_of(int softplus, M raw, float bias) {
    const float v = widen(raw) + bias;
    return softplus ? softplus_f(v) : v;
}
template <int COUNT, typename M>
__device__ __forceinline__ void steps_of(float (&d)[COUNT], int softplus, const M (&raw)[COUNT], float bias) {
    if (softplus) {                     // the branch outside: what a block knows of its values saves operations
#pragma unroll
        for (int j = 0; j < COUNT; ++j) d[j] = softplus_f(widen(raw[j]) + bias);
    } else {
#pragma unroll
        for (int j = 0; j < COUNT; ++j) d[j] = widen(raw[j]) + bias;
    }
}

// base[c] with the row in scalar registers and the lane's share as a 32-bit byte offset: one memory instruction
// without address arithmetic.
template <typename M>
__device__ __forceinline__ M& lane_at(M* base, unsigned lane_bytes) {
    using Byte = std::conditional_t<std::is_const<M>::value, const char, char>;
    return *reinterpret_cast<M*>(reinterpret_cast<Byte*>(base) + lane_bytes);
}

// The next rows of a wavefront's channels, loaded while the ones before them are worked on.  The row is in
// scalar registers, the lane adds its channel.
constexpr int AHEAD = 4;
template <typename M, bool BACK>
struct Ahead {
    M u[AHEAD], delta[AHEAD], dy[BACK ? AHEAD : 1];
    // rows t .. t + 3 of the chunk at r0, its last one instead of those behind it, at the lane's byte offset
    __device__ __forceinline__ void load(const Scan& a, int64_t r0, int t, int len, unsigned at) {
        asm volatile("" : "+v"(at));       // hoisted out of the loop, the offset becomes 64 bits wide and is added by the lanes
        const M* pu = static_cast<const M*>(a.u) + (r0 + t) * a.u_stride;
        const M* pd = static_cast<const M*>(a.delta) + (r0 + t) * a.delta_stride;
        const M* py = BACK ? static_cast<const M*>(a.dy) + (r0 + t) * a.dy_stride : nullptr;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            u[j] = lane_at(pu, at);
            delta[j] = lane_at(pd, at);
            if (BACK) dy[j] = lane_at(py, at);
            if (t + j + 1 < len) {
                pu += a.u_stride;
                pd += a.delta_stride;
                if (BACK) py += a.dy_stride;
            }
        }
    }
};

// Channels of one workgroup of the kernels with a lane per channel: whole wavefronts, spread evenly over as
// few workgroups of at most four wavefronts as a group of channels needs.
inline int scan_block(int per) {
    const int waves = (int)ceil_div(per, WAVE), blocks = (int)ceil_div(waves, 4);
    return WAVE * (int)ceil_div(waves, blocks);
}

// One row of B or C in LDS, read by all lanes at once.
template <int NP, int SIZE>
__device__ __forceinline__ void row_of(float (&v)[SIZE], const float* p) {
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p + n);
        v[n] = q.x; v[n + 1] = q.y; v[n + 2] = q.z; v[n + 3] = q.w;
    }
}

// `state` columns from src on, padded with zeros.
template <typename M, int NP>
__device__ __forceinline__ void stage_rows(float* lds, const M* __restrict__ src, int64_t stride, int64_t row, int count,
                                           int state) {
    for (int i = threadIdx.x; i < count * NP; i += blockDim.x) {
        const int n = i % NP;
        lds[i] = n < state ? widen(src[(row + i / NP) * stride + n]) : 0.0f;
    }
    for (int n = threadIdx.x; n < NP; n += blockDim.x) lds[ZERO_ROW * NP + n] = 0.0f;
}

// A channel's states from n0 on in an (sequence, channel, n) array; zeros without the array.  Rarely run inside the
// loop over rows: the opaque offset and count keep the compiler from holding its sixteen addresses and lane masks in
// registers throughout.
template <int NP>
__device__ __forceinline__ void load_state(float (&v)[NP], const float* from, const Scan& a, int s, int c, int n0) {
#pragma unroll
    for (int n = 0; n < NP; ++n) v[n] = 0.0f;
    if (!from) return;
    int64_t at = ((int64_t)s * a.channels + c) * a.state + n0;
    int count = a.state - n0;
    asm volatile("" : "+v"(at), "+s"(count));
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const float x = from[at + min(n, count - 1)];
        v[n] = n < count ? x : 0.0f;
    }
}
template <int NP>
__device__ __forceinline__ void store_state(float* to, const float (&v)[NP], const Scan& a, int s, int c) {
    int64_t at = ((int64_t)s * a.channels + c) * a.state;
    int count = a.state;
    asm volatile("" : "+v"(at), "+s"(count));
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < count) to[at + n] = v[n];
}

template <int NP>
__device__ __forceinline__ void load_rates(float (&A2)[NP], const Scan& a, int c, int n0) {
#pragma unroll
    for (int n = 0; n < NP; ++n) A2[n] = n0 + n < a.state ? rate_of(a.A[(int64_t)c * a.state + n0 + n]) : 0.0f;
}

// Pass 1.  A lane holds a channel and up to sixteen of its states (they are independent here: more of them are
// more workgroups); B and C come from LDS.  With the reverse part a lane holds eight: its four tables of sixteen would
// not fit the registers of four wavefronts per SIMD (12007 x 2048 x 16 in bfloat16: 137 us, 92 us without).
template <typename T, int NP, bool BACK>
__global__ __launch_bounds__(256) void k_scan_sum(const Scan a) {
    using M = typename T::mem;
    __shared__ float sB[(SCAN_TILE + 1) * NP], sC[BACK ? (SCAN_TILE + 1) * NP : 1];
    const int slices = (a.state + NP - 1) / NP, n_blocks = a.groups * a.blocks_per_group * slices;
    const int sb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int cb = sb / slices, n0 = sb % slices * NP;
    const int g = cb / a.blocks_per_group;
    const int in_group = (cb % a.blocks_per_group) * blockDim.x + threadIdx.x;
    const bool live = in_group < a.per;
    const int c = g * a.per + (live ? in_group : 0);
    const int64_t r0 = (int64_t)k * a.chunk;
    const int len = (int)min((int64_t)a.chunk, a.rows - r0);
    const M* B = static_cast<const M*>(a.B) + (int64_t)g * a.state + n0;
    const M* C = static_cast<const M*>(a.C) + (int64_t)g * a.state + n0;
    const float bias = a.bias ? a.bias[c] : 0.0f;

    float A2[NP], h[NP], P[NP], R[NP];
    load_rates<NP>(A2, a, c, n0);
#pragma unroll
    for (int n = 0; n < NP; ++n) { h[n] = 0.0f; P[n] = 1.0f; R[n] = 0.0f; }
    float sum = 0.0f;
    int reset = 0;                 // a sequence start was passed: the reverse part is complete

    Ahead<M, BACK> next;
    unsigned lane_bytes = (unsigned)c * sizeof(M);       // below 2^26 (2^24 channels)
    next.load(a, r0, 0, len, lane_bytes);
    Stretch q = find_stretch(a.off, a.n_seqs, a.rows, r0, 0, len);
    for (int t0 = 0; t0 < len; t0 += SCAN_TILE) {
        const int t1 = min(t0 + SCAN_TILE, len);
        __syncthreads();
        stage_rows<M, NP>(sB, B, a.B_stride, r0 + t0, t1 - t0, a.state - n0);
        if (BACK) stage_rows<M, NP>(sC, C, a.C_stride, r0 + t0, t1 - t0, a.state - n0);
        __syncthreads();
        for (int t = t0; t < t1;) {
            if (t >= q.until) q = find_stretch(a.off, a.n_seqs, a.rows, r0, t, len);
            const int t2 = uniform(min(t1, q.until));
            if (!q.inside || q.first) {
                reset = uniform(1);
                sum = 0.0f;
                load_state<NP>(h, q.inside ? a.initial : nullptr, a, q.s, c, n0);
                q.first = false;
            }
            if (!q.inside) {
                t = t2;
                if (t < len) next.load(a, r0, t, len, lane_bytes);
                continue;
            }
            // rows t .. t2 in groups of four; OPEN: the reverse part still runs
            auto advance = [&](auto open) {
                constexpr bool OPEN = decltype(open)::value;
                while (t < t2) {
                    const int from = t, count = uniform(min(AHEAD, t2 - t));
                    const Ahead<M, BACK> now = next;
                    t = uniform(t + count);
                    if (t < len) next.load(a, r0, t, len, lane_bytes);
                    float d[AHEAD], du[AHEAD], dv[AHEAD];
                    steps_of<AHEAD>(d, a.softplus, now.delta, bias);
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j) {
                        du[j] = d[j] * widen(now.u[j]);
                        dv[j] = OPEN ? widen(now.dy[j]) : 0.0f;
                    }
                    if (count < AHEAD) {                   // rows behind the last: a step of zero changes nothing
#pragma unroll
                        for (int j = 1; j < AHEAD; ++j)
                            if (j >= count) d[j] = du[j] = dv[j] = 0.0f;
                    }
                    int at = (from - t0) * NP;
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j) {
                        float b[NP], cc[OPEN ? NP : 4];
                        row_of<NP>(b, sB + at);
                        if (OPEN) row_of<NP>(cc, sC + at);
                        at = j + 1 < count ? at + NP : ZERO_ROW * NP;
#pragma unroll
                        for (int n = 0; n < NP; ++n) {
                            const float e = exp2_hw(d[j] * A2[n]);
                            if (OPEN) {
                                P[n] *= e;
                                R[n] = fmaf(P[n], cc[n] * dv[j], R[n]);
                            }
                            h[n] = fmaf(e, h[n], du[j] * b[n]);
                        }
                        after(at, h[NP / 2]);
                    }
                    sum += (d[0] + d[1]) + (d[2] + d[3]);
                }
            };
            if (BACK && !reset) advance(std::integral_constant<bool, BACK>{});
            else advance(std::false_type{});
            if (BACK && a.dfinal && !reset && q.last && t == q.until) {   // the gradient of the state left behind enters here
                float g_end[NP];
                load_state<NP>(g_end, a.dfinal, a, q.s, c, n0);
#pragma unroll
                for (int n = 0; n < NP; ++n) R[n] = fmaf(P[n], g_end[n], R[n]);
            }
        }
    }
    if (!live) return;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n0 + n < a.state) {
            const int64_t at = ((int64_t)k * a.state + n0 + n) * a.channels + c;
            a.hst[at] = h[n];
            if (BACK) a.gst[at] = R[n];
        }
    if (n0) return;
    a.dsum[(int64_t)k * a.channels + c] = sum;
    if (c == 0) a.reset[k] = reset;
}

// Pass 2, in place: hst[k] (and, from the right, gst[k]) becomes the state that enters chunk k.  64 columns
// by 16 segments of the chunks: each segment's own composition, then the ones before it, then the segment.
// BATCH chunks are loaded at a time: one after the other they are a chain of memory latencies.  Bound by memory:
// 128 chunks of 2048 x 16 states read and written in 11 us (3.1 TB/s).
template <typename T, int BATCH>
__global__ __launch_bounds__(1024) void k_scan_carry(const Scan a) {
    __shared__ float sD[16][64], sH[16][64];
    const int lane = threadIdx.x & 63, seg = threadIdx.x >> 6;
    const bool right = blockIdx.y == 1;
    float* st = right ? a.gst : a.hst;
    const int64_t m = (int64_t)a.state * a.channels;
    const int64_t e = (int64_t)blockIdx.x * 64 + lane;
    const bool live = e < m;
    const int n = live ? (int)(e / a.channels) : 0, c = live ? (int)(e % a.channels) : 0;
    const float A2 = rate_of(a.A[(int64_t)c * a.state + n]);
    const int len = (a.n_chunks + 15) / 16;
    const int k0 = min(seg * len, a.n_chunks), k1 = min(k0 + len, a.n_chunks);
    float v[BATCH], dec[BATCH];
    int cut[BATCH];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int i = min(i0 + j, k1 - 1), k = right ? a.n_chunks - 1 - i : i;
            v[j] = live ? st[k * m + e] : 0.0f;
            dec[j] = a.dsum[(int64_t)k * a.channels + c];
            cut[j] = a.reset[k];
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) dec[j] = exp2_hw(A2 * dec[j]);
    };
    float D = 1.0f, H = 0.0f;
    for (int i0 = k0; i0 < k1; i0 += BATCH) {
        fetch(i0);
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (i0 + j < k1) {
                H = cut[j] ? v[j] : fmaf(dec[j], H, v[j]);
                D = cut[j] ? -1.0f : D * dec[j];           // the sign, which no decay changes, says that there was a cut
            }
    }
    sD[seg][lane] = D; sH[seg][lane] = H;
    __syncthreads();
    float carry = 0.0f;
    // what comes before a cut does not pass it; what comes before decays whose product is zero does, if it is a NaN
    for (int s = 0; s < seg; ++s) carry = signbit(sD[s][lane]) ? sH[s][lane] : fmaf(sD[s][lane], carry, sH[s][lane]);
    for (int i0 = k0; i0 < k1; i0 += BATCH) {
        if (len > BATCH) fetch(i0);                    // a shorter segment is still in registers
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (i0 + j < k1) {
                const int k = right ? a.n_chunks - 1 - (i0 + j) : i0 + j;
                if (live) st[k * m + e] = carry;
                carry = cut[j] ? v[j] : fmaf(dec[j], carry, v[j]);
            }
    }
}

// Pass 3: y, and the states that sequences leave behind.  A lane holds a channel with all its states, so that the sum
// over them needs no other lane.  Four rows of u and delta are in flight; 150 us at 16384 x 2048 x 16 in bfloat16.
template <typename T, int NP>
__global__ __launch_bounds__(256) void k_scan_fwd(const Scan a) {
    using M = typename T::mem;
    __shared__ float sB[(SCAN_TILE + 1) * NP], sC[(SCAN_TILE + 1) * NP];
    const int n_blocks = a.groups * a.blocks_per_group;
    const int cb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int g = cb / a.blocks_per_group;
    const int in_group = (cb % a.blocks_per_group) * blockDim.x + threadIdx.x;
    const bool live = in_group < a.per;
    const int c = g * a.per + (live ? in_group : 0);
    const int64_t r0 = (int64_t)k * a.chunk;
    const int len = (int)min((int64_t)a.chunk, a.rows - r0);
    M* y = static_cast<M*>(a.y);
    const M* B = static_cast<const M*>(a.B) + (int64_t)g * a.state;
    const M* C = static_cast<const M*>(a.C) + (int64_t)g * a.state;
    const float bias = a.bias ? a.bias[c] : 0.0f;
    const float skip = a.D ? a.D[c] : 0.0f;

    float A2[NP], h[NP];
    load_rates<NP>(A2, a, c, 0);
#pragma unroll
    for (int n = 0; n < NP; ++n)
        h[n] = a.n_chunks > 1 && n < a.state ? a.hst[((int64_t)k * a.state + n) * a.channels + c] : 0.0f;

    Ahead<M, false> next;
    unsigned lane_bytes = (unsigned)c * sizeof(M);       // below 2^26 (2^24 channels)
    next.load(a, r0, 0, len, lane_bytes);
    Stretch q = find_stretch(a.off, a.n_seqs, a.rows, r0, 0, len);
    for (int t0 = 0; t0 < len; t0 += SCAN_TILE) {
        const int t1 = min(t0 + SCAN_TILE, len);
        __syncthreads();
        stage_rows<M, NP>(sB, B, a.B_stride, r0 + t0, t1 - t0, a.state);
        stage_rows<M, NP>(sC, C, a.C_stride, r0 + t0, t1 - t0, a.state);
        __syncthreads();
        for (int t = t0; t < t1;) {
            if (t >= q.until) q = find_stretch(a.off, a.n_seqs, a.rows, r0, t, len);
            const int t2 = uniform(min(t1, q.until));
            if (!q.inside) {
                if (a.zero_rest && live)
                    for (int i = t; i < t2; ++i) lane_at(y + (r0 + i) * a.y_stride, lane_bytes) = narrow<M>(0.0f);
                t = t2;
                if (t < len) next.load(a, r0, t, len, lane_bytes);
                continue;
            }
            if (q.first) {
                load_state<NP>(h, a.initial, a, q.s, c, 0);
                q.first = false;
            }
            while (t < t2) {
                const int from = t, count = uniform(min(AHEAD, t2 - t));
                const Ahead<M, false> now = next;
                t = uniform(t + count);
                if (t < len) next.load(a, r0, t, len, lane_bytes);
                float d[AHEAD], du[AHEAD], out[AHEAD];
                steps_of<AHEAD>(d, a.softplus, now.delta, bias);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const float uv = widen(now.u[j]);
                    du[j] = d[j] * uv;
                    out[j] = skip * uv;
                }
                if (count < AHEAD) {                       // rows behind the last: a step of zero changes nothing
#pragma unroll
                    for (int j = 1; j < AHEAD; ++j)
                        if (j >= count) d[j] = du[j] = 0.0f;
                }
                if (!a.D) {                                // no term at all, also where u is infinite
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j) out[j] = 0.0f;
                }
                int at = (from - t0) * NP;
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    float b[NP], cc[NP];
                    row_of<NP>(b, sB + at);
                    row_of<NP>(cc, sC + at);
                    at = j + 1 < count ? at + NP : ZERO_ROW * NP;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        h[n] = fmaf(exp2_hw(d[j] * A2[n]), h[n], du[j] * b[n]);
                        out[j] = fmaf(cc[n], h[n], out[j]);
                    }
                    asm volatile("" : "+v"(out[j]));       // the sum is made here, not at the store (registers)
                    after(at, h[NP / 2]);
                }
                if (live) {
                    asm volatile("" : "+v"(lane_bytes));
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j)
                        if (j < count) lane_at(y + (r0 + from + j) * a.y_stride, lane_bytes) = narrow<M>(out[j]);
                }
            }
            if (a.final && q.last && t == q.until && live) store_state<NP>(a.final, h, a, q.s, c);
        }
    }
}

// Sequences without rows (and those whose offsets do not lie within the rows): the state passes through,
// and so does its gradient.  A workgroup takes the elements first, first + step, ... of sequence s.
struct Empties { const int64_t* off; int64_t rows, size; const float* from; float* to; };
__device__ __forceinline__ void pass_through(const Empties& a, int64_t s, int64_t first, int64_t step) {
    const int64_t start = a.off ? a.off[s] : 0, end = a.off ? min(a.off[s + 1], a.rows) : a.rows;
    if (start >= 0 && start < end) return;
    for (int64_t i = first; i < a.size; i += step) a.to[s * a.size + i] = a.from ? a.from[s * a.size + i] : 0.0f;
}
template <typename T>
__global__ __launch_bounds__(1024) void k_scan_empty(const Empties a) {
    pass_through(a, blockIdx.x, threadIdx.x, 1024);
}

// ---- gradients ---------------------------------------------------------------------------------------
// A lane holds four of a channel's states (LPC = NP / 4 lanes per channel), a workgroup of four wavefronts
// 4 * 64 / LPC channels of one group and one chunk of rows.  The chunk's d, u and dy lie in LDS by channel (eight
// rows of a channel are one or two 16-byte reads; the padding spreads sixteen channels over all banks), B and C by
// row.  The chunk is swept once forward, keeping the state at every eighth row, and then eight rows at a time
// from its end: forward again with all eight states and decays in registers, and back over them.
//   g = C dy + G;  dC = dy h;  dB = d u g;  G = a g;  w = G h_before;  dA += d w;
//   du = d sum(g B) + D dy;  dd = u sum(g B) + sum(A w)
// Eight rows without the start or end of a sequence (nearly all) run without a branch, so that LDS and exp
// latencies overlap.  Sums over n stay in the LPC lanes of a channel; dB and dC are summed over the channels of the
// wavefront (v_permlane swaps halve eight values to two, then rotations within a row of lanes), over the four
// wavefronts in LDS, and over the workgroups of a group by k_scan_reduce: a fixed order throughout.
// Bound by vector issue: 118 instructions per wavefront and row (256 elements), eight of them an exp, 29 % of them issued in
// pairs: 109 slots, 76 % of those of busy CUs (an exp takes two).  12007 x 2048 x 16 in bfloat16: 405-417 us.
constexpr int SUB = 8;

template <int NP> constexpr int bwd_lpc() { return NP / 4; }
template <int NP> constexpr int bwd_channels() { return 4 * WAVE / bwd_lpc<NP>(); }
template <int NP> constexpr int bwd_rows() { return bwd_channels<NP>() >= 256 ? 16 : bwd_channels<NP>() >= 128 ? 32 : 64; }

// Wavefronts per SIMD that the LDS of the gradient kernel allows; held to three in registers too (a few spilled
// around the rare paths) it is 8 % faster than with two.
template <typename T, int NP> constexpr int bwd_waves() { return sizeof(typename T::mem) == 2 && NP >= 16 ? 3 : 2; }

template <int LPC>
__device__ __forceinline__ float sum_states(float v) {       // over the LPC neighbouring lanes of a channel
    if (LPC >= 2) v += dpp<0xB1>(v);                          // quad_perm [1, 0, 3, 2]
    if (LPC >= 4) v += dpp<0x4E>(v);                          // quad_perm [2, 3, 0, 1]
    if (LPC >= 8) v += dpp<0x141>(v);                         // row_half_mirror
    if (LPC >= 16) v += dpp<0x140>(v);                        // row_mirror
    return v;
}

// Over the lanes of a row of 16 with equal lane % LPC, the same bits in all of them: by 8 first, so that after every
// step the values repeat at the next distance and the rotation adds the same two of them in either lane.
template <int LPC>
__device__ __forceinline__ float sum_channels(float v) {
    if (LPC <= 8) v += dpp<0x128>(v);                         // row_ror:8, 4, 2, 1
    if (LPC <= 4) v += dpp<0x124>(v);
    if (LPC <= 2) v += dpp<0x122>(v);
    if (LPC <= 1) v += dpp<0x121>(v);
    return v;
}

// Eight neighbouring elements in LDS, 16 bytes aligned.
template <typename M> struct alignas(16) Eight { Raw<M, SUB> r; };

template <typename T, int NP, int MAXR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(bwd_waves<T, NP>()))) void k_scan_bwd(const Scan a) {
    using M = typename T::mem;
    constexpr int LPC = bwd_lpc<NP>(), CPW = WAVE / LPC, CPB = 4 * CPW, NSUB = MAXR / SUB;
    constexpr int SD = MAXR + 4, SM = MAXR + 16 / (int)sizeof(M);      // distance between channels
    constexpr int QUADS = CPB / 4, PASS_ROWS = 256 / QUADS, PASSES = (MAXR + PASS_ROWS - 1) / PASS_ROWS;   // staging: four channels a thread
    __shared__ alignas(16) float sd[CPB * SD];           // d, later the gradient of d
    __shared__ alignas(16) M su[CPB * SM];               // u, later its gradient
    __shared__ alignas(16) M sdy[CPB * SM];
    __shared__ alignas(16) float sB[MAXR * NP], sC[MAXR * NP];
    constexpr int SLAB = 4 * SUB * 2 * NP;               // eight rows of dB and dC from each wavefront, twice
    __shared__ alignas(16) float slab[2 * SLAB > PASS_ROWS * CPB ? 2 * SLAB : PASS_ROWS * CPB];
    __shared__ int sseq[WAVE], sflag[WAVE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_blocks = a.groups * a.blocks_per_group;
    const int cb = blockIdx.x % n_blocks, k = blockIdx.x / n_blocks;
    const int g = cb / a.blocks_per_group, gb = cb % a.blocks_per_group;
    const int64_t r0 = (int64_t)k * a.chunk;
    const int len = (int)min((int64_t)a.chunk, a.rows - r0);
    const int c_base = g * a.per + gb * CPB, n_ch = min(a.per - gb * CPB, CPB);
    enum { OUT = 4, START = 1, END = 2, NONE = 8 };

    if (tid < WAVE) {
        int flag = NONE;
        if (tid < len) {
            const Place q = find_row(a.off, a.n_seqs, a.rows, r0 + tid);
            sseq[tid] = q.s;
            flag = !q.inside ? (OUT | START | END)
                             : (r0 + tid == q.start ? START : 0) | (r0 + tid + 1 == q.end ? END : 0);
        }
        sflag[tid] = flag;
    }
    __syncthreads();
    const int sq = (tid % QUADS) * 4, srow = tid / QUADS, s_n = max(n_ch - sq, 0);      // the thread's channels and row
    // sums over the rows of a value per channel, from the threads' shares
    auto fold = [&](const float (&v)[4], float* part) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) slab[srow * CPB + sq + i] = v[i];
        __syncthreads();
        if (part && tid < n_ch) {
            float s = 0.0f;
            for (int i = 0; i < PASS_ROWS; ++i) s += slab[i * CPB + tid];
            part[(int64_t)k * a.channels + c_base + tid] = s;
        }
        __syncthreads();
    };
    {   // rows outside every sequence count as zero, whatever they hold
        float raw[PASSES][4], uv[PASSES][4], dv[PASSES][4], bias[4], dD[4] = {};
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int64_t row = r0 + min(p * PASS_ROWS + srow, len - 1);
            load_vec<M, 4>(raw[p], static_cast<const M*>(a.delta) + row * a.delta_stride + c_base + sq, s_n);
            load_vec<M, 4>(uv[p], static_cast<const M*>(a.u) + row * a.u_stride + c_base + sq, s_n);
            load_vec<M, 4>(dv[p], static_cast<const M*>(a.dy) + row * a.dy_stride + c_base + sq, s_n);
        }
        load_vec<float, 4>(bias, a.bias + c_base + sq, a.bias ? s_n : 0);
        for (int i = tid; i < len * LPC; i += 256) {
            const int t = i / LPC, n = i % LPC * 4, count = sflag[t] & OUT ? 0 : max(a.state - n, 0);
            float b[4], cc[4];
            load_vec<M, 4>(b, static_cast<const M*>(a.B) + (r0 + t) * a.B_stride + (int64_t)g * a.state + n, count);
            load_vec<M, 4>(cc, static_cast<const M*>(a.C) + (r0 + t) * a.C_stride + (int64_t)g * a.state + n, count);
            *reinterpret_cast<float4*>(sB + i * 4) = make_float4(b[0], b[1], b[2], b[3]);
            *reinterpret_cast<float4*>(sC + i * 4) = make_float4(cc[0], cc[1], cc[2], cc[3]);
        }
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int t = p * PASS_ROWS + srow;
            const bool in = t < len && !(sflag[t] & OUT);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool has = in && i < s_n;
                const float d = has ? step_of(a.softplus, narrow<M>(raw[p][i]), bias[i]) : 0.0f;
                const float x = has ? uv[p][i] : 0.0f, y = has ? dv[p][i] : 0.0f;
                dD[i] = fmaf(x, y, dD[i]);
                if (t < MAXR) {
                    sd[(sq + i) * SD + t] = d;
                    su[(sq + i) * SM + t] = narrow<M>(x);
                    sdy[(sq + i) * SM + t] = narrow<M>(y);
                }
            }
        }
        fold(dD, a.part_D);
    }

    const int nq = lane % LPC, chl = wave * CPW + lane / LPC;       // the lane's states and channel
    const bool live = chl < n_ch;
    const int c = c_base + (live ? chl : 0), n0 = nq * 4;
    const float skip = a.D ? a.D[c] : 0.0f;
    float A2[4], h[4], G[4], dA[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        A2[i] = n0 + i < a.state ? rate_of(a.A[(int64_t)c * a.state + n0 + i]) : 0.0f;
        const bool has = a.n_chunks > 1 && live && n0 + i < a.state;
        const int64_t at = ((int64_t)k * a.state + n0 + i) * a.channels + c;
        h[i] = has ? a.hst[at] : 0.0f;
        G[i] = has ? a.gst[at] : 0.0f;
        dA[i] = 0.0f;
    }
    const int n_left = live ? max(a.state - n0, 0) : 0;
    auto enter = [&](float (&v)[4], int t, int flag, const float* from) {       // a state of the sequence of row t
        load_vec<float, 4>(v, from + ((int64_t)sseq[t] * a.channels + c) * a.state + n0, from && !(flag & OUT) ? n_left : 0);
    };
    auto four = [&](float (&v)[4], const float* p) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    };
    // eight rows of d and u of the lane's channel
    float* const pd = sd + chl * SD;
    M* const pu = su + chl * SM;
    M* const pdy = sdy + chl * SM;
    float* const pslab = slab + (wave * SUB * 2 + (lane >> 5)) * NP + n0 + ((lane >> 4) & 1) * 2;
    const uint64_t marked = __ballot(sflag[lane] != 0);
    auto flag_at = [&](int t) { return __builtin_amdgcn_readfirstlane(sflag[t]); };

    const int n_sub = (len + SUB - 1) / SUB;
    float keep[NSUB][4];
    auto sweep = [&](auto plain, int s) {
        const Eight<float> d8 = *reinterpret_cast<const Eight<float>*>(pd + s * SUB);
        const Eight<M> u8 = *reinterpret_cast<const Eight<M>*>(pu + s * SUB);
        const float* pB = sB + s * SUB * NP + n0;
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int t = s * SUB + j;
            if (!decltype(plain)::value) {
                const int flag = flag_at(t);
                if (flag & START) enter(h, t, flag, a.initial);
            }
            float b[4];
            four(b, pB + j * NP);
            const float d = d8.r.get(j), du = d * u8.r.get(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = fmaf(exp2_hw(d * A2[i]), h[i], du * b[i]);
        }
    };
    for (int s = 0; s < n_sub; ++s) {
#pragma unroll
        for (int q = 0; q < NSUB; ++q)
            if (q == s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) keep[q][i] = h[i];
            }
        if (s + 1 == n_sub) break;
        if ((marked >> (s * SUB)) & 0xff) sweep(std::false_type{}, s);
        else sweep(std::true_type{}, s);
    }

    auto back = [&](auto plain, int s) {
        constexpr bool PLAIN = decltype(plain)::value;
        float hs[SUB + 1][4], ea[SUB][4];
        float dd[SUB] = {}, gu[SUB] = {};
        const Eight<float> d8 = *reinterpret_cast<const Eight<float>*>(pd + s * SUB);
        const Eight<M> u8 = *reinterpret_cast<const Eight<M>*>(pu + s * SUB);
        const Eight<M> y8 = *reinterpret_cast<const Eight<M>*>(pdy + s * SUB);
        int at = s * SUB * NP + n0;                      // of the lane's four B in the row, and C
#pragma unroll
        for (int i = 0; i < 4; ++i) hs[0][i] = h[i];
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int t = s * SUB + j;
            float prev[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) prev[i] = hs[j][i];
            if (!PLAIN) {
                const int flag = flag_at(t);
                if (flag & NONE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) { ea[j][i] = 1.0f; hs[j + 1][i] = 0.0f; }
                    continue;
                }
                if (flag & START) enter(prev, t, flag, a.initial);
            }
            four(b, sB + at + j * NP);
            const float d = d8.r.get(j), du = d * u8.r.get(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ea[j][i] = exp2_hw(d * A2[i]);
                hs[j + 1][i] = fmaf(ea[j][i], prev[i], du * b[i]);
            }
            if (j % 2) after(at, hs[j][0]);
        }
#pragma unroll
        for (int j = SUB - 1; j >= 0; --j) {
            const int t = s * SUB + j;
            float prev[4], b[4], cc[4], red[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) prev[i] = hs[j][i];
            int flag = 0;
            if (!PLAIN) {
                flag = flag_at(t);
                if (flag & NONE) continue;
                if (flag & START) enter(prev, t, flag, a.initial);
                if (flag & END) enter(G, t, flag, a.dfinal);
            }
            four(b, sB + at + j * NP);
            four(cc, sC + at + j * NP);
            const float d = d8.r.get(j), uv = u8.r.get(j), dv = y8.r.get(j), du = d * uv;
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
                wA = fmaf(A2[i], w, wA);
            }
            after(at, G[0]);
            if (!PLAIN && (flag & START) && a.dinitial && !(flag & OUT) && n_left > 0)
                store_vec<float, 4>(a.dinitial + ((int64_t)sseq[t] * a.channels + c) * a.state + n0, G, n_left);
            gB = sum_states<LPC>(gB);
            wA = sum_states<LPC>(wA);
            dd[j] = fmaf(uv, gB, wA * LN2);                // A = A2 ln 2
            gu[j] = fmaf(d, gB, skip * dv);
            const float w0 = halve32(red[0], red[4]), w1 = halve32(red[1], red[5]);
            const float w2 = halve32(red[2], red[6]), w3 = halve32(red[3], red[7]);
            const float v0 = sum_channels<LPC>(halve16(w0, w2)), v1 = sum_channels<LPC>(halve16(w1, w3));
            // all lanes of a row with the same states hold the same sums, bit for bit: they write one place
            *reinterpret_cast<float2*>(pslab + (s & 1) * SLAB + j * 2 * NP) = make_float2(v0, v1);
        }
        if (nq == 0) {
            Eight<float> d_out;
            Eight<M> u_out;
            d_out.r.set(dd);
            u_out.r.set(gu);
            *reinterpret_cast<Eight<float>*>(pd + s * SUB) = d_out;
            *reinterpret_cast<Eight<M>*>(pu + s * SUB) = u_out;
        }
    };
    float* const part_bc = a.part_bc + ((int64_t)gb * a.rows + r0) * a.groups * NP + (int64_t)g * NP;
    const int64_t bc_which = (int64_t)a.blocks_per_group * a.rows * a.groups * NP;
    const int bc_row = a.groups * NP;
    for (int s = n_sub - 1; s >= 0; --s) {
#pragma unroll
        for (int q = 0; q < NSUB; ++q)
            if (q == s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = keep[q][i];
            }
        if ((marked >> (s * SUB)) & 0xff) back(std::false_type{}, s);
        else back(std::true_type{}, s);
        __syncthreads();          // one is enough: the other half of the slab is written before the next
        const float* sum4 = slab + (s & 1) * SLAB;
#pragma unroll
        for (int q = 0; q < (SUB * 2 * NP + 255) / 256; ++q) {
            const int i = q * 256 + tid, j = i / (2 * NP), w = i / NP & 1;
            if (i < SUB * 2 * NP && s * SUB + j < len)
                part_bc[w * bc_which + (int64_t)(s * SUB + j) * bc_row + i % NP] =
                    (sum4[i] + sum4[SLAB / 4 + i]) + (sum4[SLAB / 2 + i] + sum4[3 * SLAB / 4 + i]);
        }
    }
    if (live) store_vec<float, 4>(a.part_A + ((int64_t)k * a.channels + c) * NP + n0, dA, 4);
    __syncthreads();
    float raw[PASSES][4], bias[4], db[4] = {};
    if (a.softplus) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
            load_vec<M, 4>(raw[p], static_cast<const M*>(a.delta) + (r0 + min(p * PASS_ROWS + srow, len - 1)) * a.delta_stride + c_base + sq, s_n);
        load_vec<float, 4>(bias, a.bias + c_base + sq, a.bias ? s_n : 0);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int t = p * PASS_ROWS + srow;
        if (t < len && s_n > 0) {
            float v[4], x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = sd[(sq + i) * SD + t];
                x[i] = widen(su[(sq + i) * SM + t]);
                if (sflag[t] & OUT) v[i] = 0.0f;
                else if (a.softplus) v[i] *= sigmoid_f(raw[p][i] + bias[i]);
                db[i] += v[i];
            }
            const int64_t at = (r0 + t) * a.channels + c_base + sq;
            store_vec<M, 4>(static_cast<M*>(a.ddelta) + at, v, s_n);
            store_vec<M, 4>(static_cast<M*>(a.du) + at, x, s_n);
        }
    }
    if (a.part_bias) fold(db, a.part_bias);
}

// The sums of the partial results, one launch for all of them and, in the blocks behind sum_blocks, for the initial
// states of sequences without rows: out[e] = sum over parts of part[p][e], of rows of
// `padded` columns of which the first `inner` are kept.  64 elements by 16 slices of the parts.  17 us for the
// 65 MB of 12007 x 2048 x 16.
struct ReduceJob {
    const float* part; void* out;
    int64_t n_part, m, first_block;
    int padded, inner, wide;             // wide: out is float32, else of the element type
};
struct ReduceJobs { ReduceJob job[5]; int count; int64_t sum_blocks; Empties empties; };

template <typename T>
__global__ __launch_bounds__(1024) void k_scan_reduce(const ReduceJobs jobs) {
    using M = typename T::mem;
    __shared__ float sh[16][64];
    if (blockIdx.x >= jobs.sum_blocks) {
        pass_through(jobs.empties, blockIdx.x - jobs.sum_blocks, threadIdx.x, 1024);
        return;
    }
    int which = 0;
    for (int i = 1; i < jobs.count; ++i)
        if (blockIdx.x >= jobs.job[i].first_block) which = i;
    const ReduceJob& job = jobs.job[which];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    // few parts: the slices take different elements instead
    const bool few = job.n_part < 64;
    const int64_t e = ((int64_t)blockIdx.x - job.first_block) * (few ? 1024 : 64) + (few ? threadIdx.x : lane);
    float s = e < job.m ? sum_strided(job.part + e, few ? 0 : slice, few ? 1 : 16, job.n_part, job.m) : 0.0f;
    if (!few) {
        sh[slice][lane] = s;
        __syncthreads();
        if (slice) return;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += sh[i][lane];
    }
    if (e >= job.m || e % job.padded >= job.inner) return;
    const int64_t at = e / job.padded * job.inner + e % job.padded;
    if (job.wide) static_cast<float*>(job.out)[at] = s;
    else static_cast<M*>(job.out)[at] = narrow<M>(s);
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
// them; a slot outside the pool gives a zero row and touches no state.  A thread has four states of a channel for
// NE entries: their loads, which need the slots alone, go out together and before the list of slots is looked
// through.  256 x 4096 x 16: 28 us, 5.0 TB/s; the look through a list of 16384 takes longer than the states.
template <typename T, int NP, int NE>
__global__ __launch_bounds__(256) void k_scan_step(const ScanStep a) {
    using M = typename T::mem;
    constexpr int LPC = NP / 4;
    const int e0 = blockIdx.y * NE;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int nq = (int)(id % LPC), n0 = nq * 4;
    const bool live = id / LPC < a.channels;
    const int c = live ? (int)(id / LPC) : 0;
    const int left = live ? max(a.state - n0, 0) : 0;           // of the lane's four states, how many exist
    int slot[NE];
    bool in_pool[NE], again[NE] = {}, skipped[NE] = {};
    int64_t at[NE];
    float h[NE][4], A2[4], uv[NE], d[NE], b[NE][4], cv[NE][4];
    M raw[NE];
    const int64_t bc = (int64_t)(c / a.per) * a.state + n0;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        const int e = min(e0 + k, a.batch - 1);
        slot[k] = a.slots ? a.slots[e] : e;
        in_pool[k] = (unsigned)slot[k] < (unsigned)a.n_slots && e0 + k < a.batch;
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        at[k] = ((int64_t)(in_pool[k] ? slot[k] : 0) * a.channels + c) * a.state + n0;
        load_vec<float, 4>(h[k], a.state_in + at[k], in_pool[k] ? left : 0);
    }
    auto token = [&](int k, int e) {                            // the inputs of entry e
        uv[k] = widen(static_cast<const M*>(a.u)[(int64_t)e * a.u_stride + c]);
        raw[k] = static_cast<const M*>(a.delta)[(int64_t)e * a.delta_stride + c];
        load_vec<M, 4>(b[k], static_cast<const M*>(a.B) + (int64_t)e * a.B_stride + bc, left);
        load_vec<M, 4>(cv[k], static_cast<const M*>(a.C) + (int64_t)e * a.C_stride + bc, left);
    };
#pragma unroll
    for (int k = 0; k < NE; ++k) token(k, min(e0 + k, a.batch - 1));
    load_vec<float, 4>(A2, a.A + (int64_t)c * a.state + n0, left);
    const float bias = a.bias ? a.bias[c] : 0.0f, skip = a.D ? a.D[c] : 0.0f;
    if (a.slots) slot_use<NE>(skipped, again, a.slots, a.batch, e0, slot);
#pragma unroll
    for (int n = 0; n < 4; ++n) A2[n] = rate_of(A2[n]);
    M* y = static_cast<M*>(a.y) + c;
    auto advance = [&](int k, int e) {
        d[k] = step_of(a.softplus, raw[k], bias);
        float acc = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            h[k][n] = fmaf(exp2_hw(d[k] * A2[n]), h[k][n], d[k] * uv[k] * b[k][n]);
            acc = fmaf(cv[k][n], h[k][n], acc);
        }
        acc = sum_states<LPC>(acc);
        if (a.D) acc = fmaf(skip, uv[k], acc);
        if (live && nq == 0) y[(int64_t)e * a.y_stride] = narrow<M>(acc);
    };
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        if (e0 + k >= a.batch) break;
        if (!in_pool[k]) {
            if (live && nq == 0) y[(int64_t)(e0 + k) * a.y_stride] = narrow<M>(0.0f);
            continue;
        }
        if (skipped[k]) continue;
        advance(k, e0 + k);
        if (again[k])
            for (int e = e0 + k + 1; e < a.batch; ++e)
                if (a.slots[e] == slot[k]) {
                    token(k, e);
                    advance(k, e);
                }
        if (left > 0) store_vec<float, 4>(a.state_out + at[k], h[k], left);
    }
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

constexpr int sum_states(bool back) { return back ? 8 : 16; }
inline int sum_slices(int state, bool back) { return (int)ceil_div(state, sum_states(back)); }

// Rows per chunk of the forward pass.  A chunk costs 16 bytes per state of traffic between the passes, so
// long ones are preferred while they leave about four wavefronts for every SIMD (256 CUs x 4).  Smaller problems
// are bound by the time of one wavefront, which goes with its rows (0.6 us each), and take shorter chunks; up to
// 32 rows one pass is faster than three launches.  With 16 rows throughout, 128 throughout, and so: 1187 x 518 x 16
// 28, 103 and 28 us, 12007 x 2048 x 16 248, 197 and 193 us, 300 x 256 x 16, where so is 8, 25, 103 and 20 us.
inline int scan_fwd_chunk(const mfcc_scan_args* a) {
    if (a->rows <= 32) return 32;
    const int64_t waves = (int64_t)a->groups * ceil_div(a->channels / a->groups, WAVE);
    for (int chunk : {256, 128, 64})
        if (waves * ceil_div(a->rows, chunk) >= 4 * 1024) return chunk;
    if (waves * ceil_div(a->rows, 32) >= 768) return 32;
    return waves * ceil_div(a->rows, 16) >= 512 ? 16 : 8;
}

// Rows per chunk of the gradients, by the same trade.  16 rows throughout, as many as fit, and so: 1187 x 518 x 16
// 43, 66 and 43 us; 12007 x 2048 x 16 680, 534 and 534 us; 300 x 256 x 16, where so is 8: 29, 62 and 27 us.
inline int bwd_channels_of(int np) { return 4 * WAVE / (np / 4); }
inline int scan_bwd_chunk(const mfcc_scan_args* a) {
    const int cpb = bwd_channels_of(padded_state(a->state)), most = cpb >= 256 ? 16 : cpb >= 128 ? 32 : 64;
    const int64_t blocks = (int64_t)a->groups * ceil_div(a->channels / a->groups, cpb);
    int chunk = most;
    while (chunk > 16 && blocks * ceil_div(a->rows, chunk) < 1024) chunk /= 2;
    return blocks * ceil_div(a->rows, 16) < 512 ? 8 : chunk;
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

// The sequences that pass_through has to look at: all of them, or none.
inline int scan_empties(const mfcc_scan_args* a, const float* from, float* to, Empties* e) {
    if (!to || (!a->d_offsets && a->rows > 0)) return 0;
    *e = {a->d_offsets, a->rows, (int64_t)a->channels * a->state, from, to};
    return a->n_seqs;
}

// A launch numbers at most 2^32 - 1 threads; every limit is looked at before the first launch of a call.
inline int too_large() { return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it"); }
inline int64_t carry_blocks(const Scan& f) { return ceil_div((int64_t)f.state * f.channels, 64); }

template <typename T>
void launch_carry(const Scan& f, unsigned directions, hipStream_t st) {
    const dim3 grid((unsigned)carry_blocks(f), directions);
    // 1187 x 518 x 16 (75 chunks) 7 and 11 us; 2500 x 700 (157) 16 and 13, 12007 x 2048 (188) 34 and 29 us
    if (f.n_chunks <= 16 * 8) hipLaunchKernelGGL((k_scan_carry<T, 8>), grid, dim3(1024), 0, st, f);
    else hipLaunchKernelGGL((k_scan_carry<T, 16>), grid, dim3(1024), 0, st, f);
}

template <typename T>
int scan_forward(const mfcc_scan_args* a, hipStream_t st) {
    Scan f = scan_args(a, false);
    const int block = scan_block(f.per);
    f.blocks_per_group = (int)ceil_div(f.per, block);
    const int64_t grid = (int64_t)f.groups * f.blocks_per_group * f.n_chunks;
    if (grid > 0x7fffff || (a->d_final && a->n_seqs > 0x3fffff)) return too_large();
    if (f.n_chunks > 1 && (grid * sum_slices(f.state, false) > 0x7fffff || carry_blocks(f) > 0x3fffff)) return too_large();
    if (a->rows > 0) {
        const int rc = by_state(a->state, [&](auto np) {
            constexpr int NP = decltype(np)::value;
            if (f.n_chunks > 1) {
                hipLaunchKernelGGL((k_scan_sum<T, std::min(NP, sum_states(false)), false>), dim3((unsigned)(grid * sum_slices(f.state, false))),
                                   dim3(block), 0, st, f);
                launch_carry<T>(f, 1, st);
            }
            hipLaunchKernelGGL((k_scan_fwd<T, NP>), dim3((unsigned)grid), dim3(block), 0, st, f);
            PACKED_LAUNCHED();
            return (int)MFCC_OK;
        });
        if (rc) return rc;
    }
    Empties e;
    if (const int seqs = scan_empties(a, a->d_initial, a->d_final, &e)) {
        hipLaunchKernelGGL(k_scan_empty<T>, dim3((unsigned)seqs), dim3(1024), 0, st, e);
        PACKED_LAUNCHED();
    }
    return MFCC_OK;
}

template <typename T>
int scan_backward(const mfcc_scan_args* a, hipStream_t st) {
    using M = typename T::mem;
    Scan f = scan_args(a, true);
    return by_state(a->state, [&](auto np) {
        constexpr int NP = decltype(np)::value;
        const int block = scan_block(f.per), sum_blocks_per_group = (int)ceil_div(f.per, block);
        const int64_t sum_grid = (int64_t)f.groups * sum_blocks_per_group * f.n_chunks * sum_slices(f.state, true);
        f.blocks_per_group = (int)ceil_div(f.per, bwd_channels<NP>());
        const int64_t grid = (int64_t)f.groups * f.blocks_per_group * f.n_chunks;
        const int64_t m = a->rows * f.groups * NP;
        ReduceJobs jobs = {};
        int64_t blocks = 0;
        auto reduce = [&](const float* part, int64_t n_part, int64_t size, int padded, int inner, void* out, bool wide) {
            if (size == 0 || !out) return;
            jobs.job[jobs.count++] = {part, out, n_part, size, blocks, padded, inner, wide};
            blocks += ceil_div(size, n_part < 64 ? 1024 : 64);
        };
        reduce(f.part_bc, f.blocks_per_group, m, NP, f.state, a->d_dB, sizeof(M) == 4);
        reduce(f.part_bc + f.blocks_per_group * m, f.blocks_per_group, m, NP, f.state, a->d_dC, sizeof(M) == 4);
        reduce(f.part_A, f.n_chunks, (int64_t)f.channels * NP, NP, f.state, a->d_dA, true);
        reduce(f.part_D, f.n_chunks, f.channels, 1, 1, a->d_dD, true);
        reduce(f.part_bias, f.n_chunks, f.channels, 1, 1, a->d_ddelta_bias, true);
        jobs.sum_blocks = blocks;
        blocks += scan_empties(a, a->d_dfinal, a->d_dinitial, &jobs.empties);
        if (grid > 0x7fffff || blocks > 0x1fffff) return too_large();
        if (f.n_chunks > 1 && (sum_grid > 0x7fffff || carry_blocks(f) > 0x3fffff)) return too_large();
        if (f.n_chunks > 1) {
            Scan g = f;
            g.blocks_per_group = sum_blocks_per_group;
            hipLaunchKernelGGL((k_scan_sum<T, std::min(NP, sum_states(true)), true>), dim3((unsigned)sum_grid), dim3(block), 0, st, g);
            launch_carry<T>(f, 2, st);
        }
        if (a->rows > 0) {
            // chunks of up to sixteen rows in a kernel with LDS and registers for as many: more workgroups per CU
            // (the gradients of 1187 x 518 x 13 in float32 61 -> 53 us)
            if (f.chunk <= 16) hipLaunchKernelGGL((k_scan_bwd<T, NP, 16>), dim3((unsigned)grid), dim3(256), 0, st, f);
            else hipLaunchKernelGGL((k_scan_bwd<T, NP, bwd_rows<NP>()>), dim3((unsigned)grid), dim3(256), 0, st, f);
            PACKED_LAUNCHED();
        }
        hipLaunchKernelGGL(k_scan_reduce<T>, dim3((unsigned)blocks), dim3(1024), 0, st, jobs);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
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
        const int64_t tiles = ceil_div((int64_t)a->channels * (NP / 4), 256);
        // Four entries per thread share A and one look through the list of slots, but are a quarter of the wavefronts.  By
        // the wavefronts of one entry per thread (entries x channels x states), one and four, in us: 4096 (512 x 256 x 8) 4.3
        // and 5.0; 16384 (1024 x 256 x 16) 9.6 and 9.1, without slots 7.9 and 8.0; 65536 (1024 x 1024 x 16) 29.3 and 28.7, without
        // slots 24.2 and 25.7; 131072 (2048 x 1024 x 16) 60.5 and 51.3, without 45.5 and 44.9, few entries (128 x 4096 x 64)
        // 54.6 and 50.2; 65536 of few entries (256 x 4096 x 16) 29.0 and 29.4.
        const int64_t waves = ceil_div((int64_t)a->channels * (NP / 4), WAVE) * f.batch;
        if (waves >= 96 * 1024 || (slots && f.batch >= 512 && waves >= 12 * 1024))
            hipLaunchKernelGGL((k_scan_step<T, NP, 4>), dim3((unsigned)tiles, (unsigned)ceil_div(f.batch, 4)), dim3(256), 0, st, f);
        else
            hipLaunchKernelGGL((k_scan_step<T, NP, 1>), dim3((unsigned)tiles, (unsigned)f.batch), dim3(256), 0, st, f);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

}  // namespace packed
