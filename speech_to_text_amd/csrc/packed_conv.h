// Short causal convolution over packed rows: forward, gradients, single tokens.
//   p[t, c] = bias[c] + sum_j w[c, j] x[t - (K - 1) + j, c],   y = p or p * sigmoid(p)
// with the rows before a sequence taken from its initial state (the K - 1 rows before it) or zero.
//
// Bound by memory: K fused multiply-adds per element against two (forward) or three (backward) rows of
// traffic.  A thread owns four neighbouring channels and walks down a tile of rows with the last K - 1 rows in
// registers, so a row is read once per tile plus K - 1 rows of overlap (from cache).  Rows are taken several at
// a time: their loads are in flight together.
#pragma once
#include "packed.h"

namespace packed {

constexpr int GROUP = 4;      // rows per step of a thread in the backward pass

struct ConvFwd {
    const void* x; int64_t x_stride;
    const float *w, *bias;
    const int64_t* off;
    const void* initial;
    void* y; int64_t y_stride;
    int64_t rows; int n_seqs, channels, n_vec, tile;
    int zero_rest, act, room;
};

// The taps and biases of the thread's channels (neighbours in memory).
template <int K, int VEC>
__device__ __forceinline__ void load_taps(float (&w)[K][VEC], float (&b)[VEC], const float* __restrict__ weight,
                                          const float* __restrict__ bias, int c0, int n) {
    float flat[VEC * K];
    load_vec<float, VEC * K>(flat, weight + (int64_t)c0 * K, n >= VEC ? VEC * K : n * K);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
        for (int j = 0; j < K; ++j) w[j][i] = flat[i * K + j];
    if (bias) load_vec<float, VEC>(b, bias + c0, n);
    else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) b[i] = 0.0f;
    }
}

// p sigmoid(p) of the forward pass and of single tokens: one function, so that tokens give the prompt's bits.  In 16-bit
// types y is all there is of it (30011 x 4096: 98 us, 101 us with sigmoid_f).
template <typename M>
__device__ __forceinline__ float silu_f(float p) {
    return p * (sizeof(M) == 4 ? sigmoid_f(p) : sigmoid_to_16(p));
}

// The value tap `back` rows before a row of sequence q reads: x, the initial state, or zero.
template <typename M, int K, int VEC>
__device__ __forceinline__ void tap_of(float (&v)[VEC], const float (&near)[VEC], const M* initial, const Place& q,
                                       int64_t row, int back, int channels, int c0, int n) {
    const int64_t at = row - back - q.start;              // row within the sequence, negative before it
    if (at >= 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = near[i];
    } else if (initial) {
        load_vec<M, VEC>(v, initial + ((int64_t)q.s * (K - 1) + (K - 1) + at) * channels + c0, n);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
    }
}

// A thread walks down its tile G rows at a time.  Waiting for memory is what bounds it, so the next G rows are in
// flight while the current ones are computed, and rows are kept in their memory type (in float32 the window and
// the rows ahead would cost half the wavefronts).  30011 x 4096, K = 4, bfloat16: 98 us, 5.0 TB/s, the rate of a copy.
template <typename T, int K, int VEC, int G>
__global__ __launch_bounds__(256) void k_conv_fwd(const ConvFwd a) {
    using M = typename T::mem;
    const unsigned id = xcd_order(blockIdx.x, gridDim.x) * 256 + threadIdx.x;      // below 2^31
    const int64_t r0 = (int64_t)(id / (unsigned)a.n_vec) * a.tile;
    const int c0 = (int)(id % (unsigned)a.n_vec) * VEC;
    if (r0 >= a.rows) return;
    const int n = a.channels - c0;
    const int64_t r1 = min(r0 + a.tile, a.rows);
    const M* x = static_cast<const M*>(a.x) + c0;
    M* y = static_cast<M*>(a.y) + c0;
    const M* initial = static_cast<const M*>(a.initial);

    Raw<M, VEC> line[K - 1 + G], next[G];
    auto fetch = [&](int64_t r) {
        const bool room = a.room && (r1 < a.rows || r + G < a.rows);
#pragma unroll
        for (int g = 0; g < G; ++g) load_raw<M, VEC>(next[g], x + min(r + g, r1 - 1) * a.x_stride, n, room);
    };
    fetch(r0);
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
        load_raw<M, VEC>(line[j], x + max(r0 - (K - 1) + j, (int64_t)0) * a.x_stride, n, a.room && a.rows > 1);
    float w[K][VEC], b[VEC];
    load_taps<K, VEC>(w, b, a.w, a.bias, c0, n);
    Place q = find_row(a.off, a.n_seqs, a.rows, r0);
    auto finish = [&](float (&acc)[VEC], int64_t row) {
        if (a.act) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = silu_f<M>(acc[i]);
        }
        store_vec<M, VEC>(y + row * a.y_stride, acc, n);
    };
    for (int64_t r = r0; r < r1; r += G) {
#pragma unroll
        for (int g = 0; g < G; ++g) line[K - 1 + g] = next[g];
        if (r + G < r1) fetch(r + G);
        if (q.inside && r >= q.start + (K - 1) && r + G <= min(q.end, r1)) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float acc[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    acc[i] = b[i];
#pragma unroll
                    for (int j = 0; j < K; ++j) acc[i] = fmaf(w[j][i], line[g + j].get(i), acc[i]);
                }
                finish(acc, r + g);
            }
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int64_t row = r + g;
                if (row >= r1) break;
                if (row >= q.until) q = find_row(a.off, a.n_seqs, a.rows, row);
                float acc[VEC];
                if (!q.inside) {
                    if (a.zero_rest) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
                        store_vec<M, VEC>(y + row * a.y_stride, acc, n);
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] = b[i];
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    float v[VEC], near[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) near[i] = line[g + j].get(i);
                    tap_of<M, K, VEC>(v, near, initial, q, row, K - 1 - j, a.channels, c0, n);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w[j][i], v[i], acc[i]);
                }
                finish(acc, row);
            }
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) line[j] = line[j + G];
    }
}

// The state a sequence leaves behind: its last K - 1 rows, the initial state standing before a short one.
// A sequence whose offsets do not lie within the rows keeps its initial state.
template <typename T>
__global__ __launch_bounds__(256) void k_conv_state(const typename T::mem* __restrict__ x, int64_t x_stride,
                                                    const int64_t* __restrict__ off, int n_seqs, int64_t rows,
                                                    int channels, int keep, const typename T::mem* __restrict__ initial,
                                                    typename T::mem* __restrict__ state) {
    using M = typename T::mem;
    const int64_t total = (int64_t)n_seqs * keep * channels;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int c = (int)(i % channels);
        const int64_t sj = i / channels;
        const int j = (int)(sj % keep);
        const int64_t s = sj / keep;
        int64_t start = off ? off[s] : 0, end = off ? min(off[s + 1], rows) : rows;
        if (start < 0 || start > end) start = end = 0;
        const int64_t at = end - start - keep + j;        // row within the sequence
        M v = (M)0.0f;
        if (at >= 0) v = x[(start + at) * x_stride + c];
        else if (initial) v = initial[(s * keep + keep + at) * channels + c];
        state[i] = v;
    }
}

struct ConvBwd {
    const void* x; int64_t x_stride;
    const void* dy; int64_t dy_stride;
    const float *w, *bias;
    const int64_t* off;
    const void *initial, *dstate;
    void* dx; int64_t dx_stride;
    float* part;                 // (row tiles / 4, K + 1, channels): sums for dweight and dbias
    void* dinitial;
    int64_t rows; int n_seqs, channels, n_vec, tile, act, room;
};

// dp = dy * act'(p) is formed for the tile's rows and the K - 1 rows behind it; dx[o] gathers the K values
// of dp that read row o, and the products dp * x add up to the tile's share of dweight.
// Three rows of traffic and 2 K registers of sums per channel: fewer wavefronts than the forward pass has.  30011 x
// 4096, K = 4: 187 us in bfloat16 (3.9 TB/s), 326 us in float32 (4.5 TB/s); 6001 x 1545, K = 3, float32: 36 us.
template <typename T, int K, int VEC>
__global__ __launch_bounds__(256) void k_conv_bwd(const ConvBwd a) {
    using M = typename T::mem;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);       // row addresses in scalar registers
    const int cv = blockIdx.x * 64 + lane;
    const int c0 = cv * VEC;
    const bool live = cv < a.n_vec;
    const int n = live ? a.channels - c0 : 0;
    const int64_t r0 = ((int64_t)blockIdx.y * 4 + wave) * a.tile;
    const int64_t r1 = min(r0 + a.tile, a.rows);
    const M* x = static_cast<const M*>(a.x) + c0;
    const M* dy = static_cast<const M*>(a.dy) + c0;
    M* dx = static_cast<M*>(a.dx) + c0;
    const M* initial = static_cast<const M*>(a.initial);
    const M* dstate = static_cast<const M*>(a.dstate);

    float dw[K][VEC] = {}, db[VEC] = {};
    if (live && r0 < a.rows) {
        float w[K][VEC], b[VEC];
        load_taps<K, VEC>(w, b, a.w, a.bias, c0, n);
        Raw<M, VEC> line[K - 1 + GROUP], dyr[GROUP], next_x[GROUP], next_dy[GROUP];
        float dp[K - 1 + GROUP][VEC];
        auto fetch = [&](int64_t r) {
            const bool room = a.room && r + GROUP < a.rows;
#pragma unroll
            for (int g = 0; g < GROUP; ++g) {
                const int64_t row = min(r + g, a.rows - 1);
                load_raw<M, VEC>(next_x[g], x + row * a.x_stride, n, room);
                load_raw<M, VEC>(next_dy[g], dy + row * a.dy_stride, n, room);
            }
        };
        fetch(r0);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            load_raw<M, VEC>(line[j], x + max(r0 - (K - 1) + j, (int64_t)0) * a.x_stride, n, a.room && a.rows > 1);
#pragma unroll
            for (int i = 0; i < VEC; ++i) dp[j][i] = 0.0f;    // rows before the tile: their dx belongs to the tile above
        }
        Place q = find_row(a.off, a.n_seqs, a.rows, r0);
        for (int64_t r = r0; r < r1 + (K - 1); r += GROUP) {
#pragma unroll
            for (int g = 0; g < GROUP; ++g) { line[K - 1 + g] = next_x[g]; dyr[g] = next_dy[g]; }
            if (r + GROUP < r1 + (K - 1)) fetch(r + GROUP);
            // the whole group, and the rows whose dx it completes, inside one sequence
            const bool plain = q.inside && r - (K - 1) >= q.start && r + GROUP <= q.end;
#pragma unroll
            for (int g = 0; g < GROUP; ++g) {
                const int64_t row = r + g;
                bool inside = true;
                if (!plain) {
                    if (row >= q.until && row < a.rows) q = find_row(a.off, a.n_seqs, a.rows, row);
                    inside = q.inside && row < a.rows && row < r1 + (K - 1);
                }
                float (&d)[VEC] = dp[K - 1 + g];
                if (inside) {
                    float tap[K][VEC];
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        float near[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) tap[j][i] = near[i] = line[g + j].get(i);
                        if (!plain) tap_of<M, K, VEC>(tap[j], near, initial, q, row, K - 1 - j, a.channels, c0, n);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        d[i] = dyr[g].get(i);
                        if (a.act) {
                            float p = b[i];
#pragma unroll
                            for (int j = 0; j < K; ++j) p = fmaf(w[j][i], tap[j][i], p);
                            const float sg = sigmoid_f(p);
                            d[i] *= sg * fmaf(p, 1.0f - sg, 1.0f);
                        }
                    }
                    if (row < r1) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            db[i] += d[i];
#pragma unroll
                            for (int j = 0; j < K; ++j) dw[j][i] = fmaf(d[i], tap[j][i], dw[j][i]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) d[i] = 0.0f;
                }
                // row o is complete: rows o .. row read it, with taps K - 1 .. 0
                const int64_t o = row - (K - 1);
                float acc[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
                if (plain) {
#pragma unroll
                    for (int j = 0; j < K; ++j)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w[K - 1 - j][i], dp[g + j][i], acc[i]);
                    if (o >= r0 && o < r1) store_vec<M, VEC>(dx + o * a.dx_stride, acc, n);
                } else if (o >= r0 && o < r1) {
                    const Place p = find_row(a.off, a.n_seqs, a.rows, o);
                    if (p.inside) {
#pragma unroll
                        for (int j = 0; j < K; ++j)
                            if (o + j < p.end) {
#pragma unroll
                                for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w[K - 1 - j][i], dp[g + j][i], acc[i]);
                            }
                        if (dstate && p.end - o <= K - 1) {
                            float s[VEC];
                            load_vec<M, VEC>(s, dstate + ((int64_t)p.s * (K - 1) + (K - 1) - (p.end - o)) * a.channels + c0, n);
#pragma unroll
                            for (int i = 0; i < VEC; ++i) acc[i] += s[i];
                        }
                    }
                    store_vec<M, VEC>(dx + o * a.dx_stride, acc, n);
                }
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                line[j] = line[j + GROUP];
#pragma unroll
                for (int i = 0; i < VEC; ++i) dp[j][i] = dp[j + GROUP][i];
            }
        }
    }
    // the four row tiles of the block, then one partial sum per block: a fixed order, the same on every run
    __shared__ float sh[4][64 * VEC];
#pragma unroll
    for (int j = 0; j <= K; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) sh[wave][i * 64 + lane] = j < K ? dw[j < K ? j : 0][i] : db[i];
        __syncthreads();
        for (int e = threadIdx.x; e < 64 * VEC; e += 256) {
            const int c = blockIdx.x * 64 * VEC + e;
            const int from = (e % VEC) * 64 + e / VEC;
            if (c < a.channels)
                a.part[((int64_t)blockIdx.y * (K + 1) + j) * a.channels + c] =
                    (sh[0][from] + sh[1][from]) + (sh[2][from] + sh[3][from]);
        }
    }
}

// Gradient of the initial state: row i of it lies K - 1 - i rows before the sequence and is read by the
// rows q <= i with tap i - q; what a short sequence hands on of it comes back from dstate.
template <typename T, int K>
__device__ __forceinline__ void conv_dinitial(const ConvBwd& a, int64_t id) {
    using M = typename T::mem;
    if (id >= (int64_t)a.n_seqs * a.channels) return;
    const int64_t s = id / a.channels;
    const int c = (int)(id % a.channels);
    int64_t start = a.off ? a.off[s] : 0, end = a.off ? min(a.off[s + 1], a.rows) : a.rows;
    if (start < 0 || start > end) start = end = 0;
    const int64_t len = end - start;
    const M* x = static_cast<const M*>(a.x) + c;
    const M* dy = static_cast<const M*>(a.dy) + c;
    const M* initial = static_cast<const M*>(a.initial);
    const M* dstate = static_cast<const M*>(a.dstate);
    float line[2 * (K - 1) + 1], w[K], di[K];             // initial rows, then the first K - 1 rows
#pragma unroll
    for (int j = 0; j < K; ++j) { w[j] = a.w[(int64_t)c * K + j]; di[j] = 0.0f; }
    const float b = a.bias ? a.bias[c] : 0.0f;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        line[j] = initial ? widen(initial[(s * (K - 1) + j) * a.channels + c]) : 0.0f;
        line[K - 1 + j] = j < len ? widen(x[(start + j) * a.x_stride]) : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < K - 1; ++q) {
        if (q >= len) break;
        float d = widen(dy[(start + q) * a.dy_stride]);
        if (a.act) {
            float p = b;
#pragma unroll
            for (int j = 0; j < K; ++j) p = fmaf(w[j], line[q + j], p);
            const float sg = sigmoid_f(p);
            d *= sg * fmaf(p, 1.0f - sg, 1.0f);
        }
#pragma unroll
        for (int i = q; i < K - 1; ++i) di[i] = fmaf(w[i - q], d, di[i]);
    }
    M* out = static_cast<M*>(a.dinitial);
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
        float v = di[i];
        if (dstate && i >= len) v += widen(dstate[(s * (K - 1) + i - len) * a.channels + c]);
        out[(s * (K - 1) + i) * a.channels + c] = narrow<M>(v);
    }
}

// dweight (channels, K) and dbias (channels) from the partial sums; the blocks from `sum_blocks` on, if any, take
// the gradient of the initial state (4 us at 6001 x 1545).
template <typename T, int K>
__global__ __launch_bounds__(1024) void k_conv_finish(const ConvBwd a, int64_t n_part, int sum_blocks,
                                                      float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float sh[16][64];
    if (blockIdx.x >= (unsigned)sum_blocks) {
        conv_dinitial<T, K>(a, (int64_t)(blockIdx.x - sum_blocks) * 1024 + threadIdx.x);
        return;
    }
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int64_t m = (int64_t)(K + 1) * a.channels;
    const int64_t e = (int64_t)blockIdx.x * 64 + lane;
    sh[slice][lane] = e < m ? sum_strided(a.part + e, slice, 16, n_part, m) : 0.0f;
    __syncthreads();
    if (slice == 0 && e < m) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += sh[i][lane];
        const int j = (int)(e / a.channels), c = (int)(e % a.channels);
        if (j < K) dweight[(int64_t)c * K + j] = v;
        else if (dbias) dbias[c] = v;
    }
}

struct ConvStep {
    const void* x; int64_t x_stride;
    const void* state; void* new_state;
    const float *w, *bias;
    const int32_t* slots;
    void* y; int64_t y_stride;
    int batch, n_slots, channels, n_vec, act;
};

// One token per entry.  Entries that name the same slot are successive tokens of that sequence: the first
// of them takes them all, in order, so no two threads touch one state.  A slot outside the pool (a padded
// entry) gives a zero row and touches no state.  Bound by the latency of one load after another: 32 x 2048 in 3.6 us.
template <typename T, int K, int VEC>
__global__ __launch_bounds__(256) void k_conv_step(const ConvStep a) {
    using M = typename T::mem;
    const int e0 = blockIdx.y;
    const int cv = blockIdx.x * 256 + threadIdx.x;
    int slot = e0;
    bool again = false;
    if (a.slots) {
        slot = a.slots[e0];
        bool before[1], after[1];
        slot_use<1>(before, after, a.slots, a.batch, e0, {slot});
        if (before[0] && (unsigned)slot < (unsigned)a.n_slots) return;
        again = after[0];
    }
    if (cv >= a.n_vec) return;
    const int c0 = cv * VEC, n = a.channels - c0;
    M* y = static_cast<M*>(a.y) + c0;
    if ((unsigned)slot >= (unsigned)a.n_slots) {
        float z[VEC] = {};
        store_vec<M, VEC>(y + (int64_t)e0 * a.y_stride, z, n);
        return;
    }
    const M* x = static_cast<const M*>(a.x) + c0;
    const M* state = static_cast<const M*>(a.state) + (int64_t)slot * (K - 1) * a.channels + c0;
    M* next = static_cast<M*>(a.new_state) + (int64_t)slot * (K - 1) * a.channels + c0;
    float w[K][VEC], b[VEC], win[K][VEC];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) load_vec<M, VEC>(win[j], state + (int64_t)j * a.channels, n);
    load_taps<K, VEC>(w, b, a.w, a.bias, c0, n);
    for (int e = e0; e < a.batch; ++e) {
        if (e != e0) {
            if (!again) break;
            if (a.slots[e] != slot) continue;
        }
        load_vec<M, VEC>(win[K - 1], x + (int64_t)e * a.x_stride, n);
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            acc[i] = b[i];
#pragma unroll
            for (int j = 0; j < K; ++j) acc[i] = fmaf(w[j][i], win[j][i], acc[i]);
            if (a.act) acc[i] = silu_f<M>(acc[i]);
        }
        store_vec<M, VEC>(y + (int64_t)e * a.y_stride, acc, n);
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) win[j][i] = win[j + 1][i];
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) store_vec<M, VEC>(next + (int64_t)j * a.channels, win[j], n);
}

// Channels of a thread.  With eight (16 bytes of a 16-bit type) the taps, sums and rows in flight cost half the
// wavefronts (125 against 98 us for 30011 x 4096 in bfloat16).
constexpr int CONV_VEC = 4;
constexpr int CONV_AHEAD = 8;      // rows in flight of the forward pass

// Rows per thread of the forward pass: a long tile reads its taps and the K - 1 rows of overlap less often, but
// below about eight wavefronts per SIMD (256 CUs x 4) the chip is not full.  16 rows throughout, 128 throughout, and
// so, K = 4, bfloat16: 600 x 512 7.8, 31 and 6.2 us; 4000 x 1024 9.2, 33 and 7.3 us; 30011 x 4096 100, 103 and 98 us.
inline int conv_fwd_tile(int64_t rows, int n_vec) {
    for (int tile : {128, 64, 32, 16})
        if (ceil_div(rows, tile) * n_vec >= 8 * 1024 * WAVE) return tile;
    return 8;
}

// Rows per wavefront of the backward pass (it also reads K - 1 rows of overlap and writes K + 1 partial sums per four
// tiles).  K = 4, bfloat16, with the summing launch, by tiles of 4, 8, 16 and 128 rows: 600 x 512 11, 13, 18, 88 us; 4000
// x 1024 21, 18, 20, 89; 12000 x 1024 40, 33, 28, 90.  By 16, 32, 64 and 128 rows: 30011 x 2048 102, 94, 94, 112 us; 30011 x
// 4096 201, 179, 187, 172; 20000 x 8192 257, 238, 232, 239: within 9 % of the best tile.
inline int conv_bwd_tile(int64_t rows, int n_vec) {
    const int64_t across = ceil_div(n_vec, WAVE);
    for (int tile : {128, 64, 32})
        if (ceil_div(rows, tile) * across >= 4 * 1024) return tile;
    const int64_t waves = ceil_div(rows, 16) * across;
    return waves >= 2048 ? 16 : waves >= 512 ? 8 : 4;
}

inline int64_t conv_bwd_parts(const mfcc_conv_args* a) {
    return ceil_div(a->rows, 4 * (int64_t)conv_bwd_tile(a->rows, (int)ceil_div(a->channels, CONV_VEC)));
}

template <typename Fn>
int by_width(int width, Fn&& fn) {
    switch (width) {
        case 1: return fn(std::integral_constant<int, 1>{});
        case 2: return fn(std::integral_constant<int, 2>{});
        case 3: return fn(std::integral_constant<int, 3>{});
        case 4: return fn(std::integral_constant<int, 4>{});
        case 5: return fn(std::integral_constant<int, 5>{});
        case 6: return fn(std::integral_constant<int, 6>{});
        case 7: return fn(std::integral_constant<int, 7>{});
        case 8: return fn(std::integral_constant<int, 8>{});
    }
    return mfcc_detail::fail(MFCC_E_INVALID, "width must lie between 1 and 8");
}

// The arguments of the three below have been checked.
template <typename T>
int conv_forward(const mfcc_conv_args* a, hipStream_t st) {
    using M = typename T::mem;
    constexpr int VEC = CONV_VEC;
    return by_width(a->width, [&](auto width) {
        constexpr int K = decltype(width)::value;
        if (a->rows > 0) {
            ConvFwd f;
            f.x = a->d_x; f.x_stride = a->x_stride; f.w = a->d_weight; f.bias = a->d_bias; f.off = a->d_offsets;
            f.initial = a->d_initial; f.y = a->d_y; f.y_stride = a->y_stride; f.rows = a->rows;
            f.n_seqs = a->n_seqs; f.channels = a->channels; f.n_vec = (int)ceil_div(a->channels, VEC);
            f.tile = conv_fwd_tile(a->rows, f.n_vec); f.zero_rest = a->zero_rest; f.act = a->activation == MFCC_ACT_SILU;
            f.room = has_room(f.x, f.x_stride, VEC);
            const int64_t blocks = ceil_div(ceil_div(a->rows, f.tile) * f.n_vec, 256);
            if (blocks > 0x7fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
            hipLaunchKernelGGL((k_conv_fwd<T, K, VEC, CONV_AHEAD>), dim3((unsigned)blocks), dim3(256), 0, st, f);
            PACKED_LAUNCHED();
        }
        if (a->d_state && a->n_seqs > 0 && K > 1) {
            const int64_t total = (int64_t)a->n_seqs * (K - 1) * a->channels;
            const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(total, 256), 65536);
            hipLaunchKernelGGL((k_conv_state<T>), dim3(blocks), dim3(256), 0, st, static_cast<const M*>(a->d_x),
                               a->x_stride, a->d_offsets, a->n_seqs, a->rows, a->channels, K - 1,
                               static_cast<const M*>(a->d_initial), static_cast<M*>(a->d_state));
            PACKED_LAUNCHED();
        }
        return (int)MFCC_OK;
    });
}

template <typename T>
int conv_backward(const mfcc_conv_args* a, hipStream_t st) {
    return by_width(a->width, [&](auto width) {
        constexpr int K = decltype(width)::value;
        ConvBwd f;
        f.x = a->d_x; f.x_stride = a->x_stride; f.dy = a->d_dy; f.dy_stride = a->dy_stride; f.w = a->d_weight;
        f.bias = a->d_bias; f.off = a->d_offsets; f.initial = a->d_initial; f.dstate = a->d_dstate; f.dx = a->d_dx;
        f.dx_stride = a->dx_stride; f.part = static_cast<float*>(a->d_workspace); f.dinitial = a->d_dinitial;
        f.rows = a->rows; f.n_seqs = a->n_seqs; f.channels = a->channels; f.act = a->activation == MFCC_ACT_SILU;
        f.n_vec = (int)ceil_div(a->channels, CONV_VEC); f.tile = conv_bwd_tile(a->rows, f.n_vec);
        f.room = has_room(f.x, f.x_stride, CONV_VEC) && has_room(f.dy, f.dy_stride, CONV_VEC);
        const int64_t parts = conv_bwd_parts(a);
        const int64_t sum_blocks = ceil_div((int64_t)(K + 1) * a->channels, 64);
        const int64_t more = a->d_dinitial && K > 1 ? ceil_div((int64_t)a->n_seqs * a->channels, 1024) : 0;
        if (parts > 65535 || sum_blocks + more > 0x1fffff) return mfcc_detail::fail(MFCC_E_UNSUPPORTED, "batch too large: split it");
        if (a->rows > 0) {
            hipLaunchKernelGGL((k_conv_bwd<T, K, CONV_VEC>), dim3((unsigned)ceil_div(f.n_vec, WAVE), (unsigned)parts),
                               dim3(256), 0, st, f);
            PACKED_LAUNCHED();
        }
        hipLaunchKernelGGL((k_conv_finish<T, K>), dim3((unsigned)(sum_blocks + more)), dim3(1024), 0, st, f, parts,
                           (int)sum_blocks, a->d_dweight, a->d_dbias);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

template <typename T>
int conv_step(ConvStep f, int width, hipStream_t st) {
    constexpr int VEC = CONV_VEC;
    return by_width(width, [&](auto w) {
        constexpr int K = decltype(w)::value;
        f.n_vec = (int)ceil_div(f.channels, VEC);
        hipLaunchKernelGGL((k_conv_step<T, K, VEC>), dim3((unsigned)ceil_div(f.n_vec, 256), (unsigned)f.batch), dim3(256), 0,
                           st, f);
        PACKED_LAUNCHED();
        return (int)MFCC_OK;
    });
}

}  // namespace packed
