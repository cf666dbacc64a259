// Group norm with an activation over channels-last data, forward and backward (custos_hip_group_norm,
// custos_hip_add_group_norm_grad in include/custos_hip.h).  No counterpart in the reference.
//
// x is [samples, positions, channels]; the channels of a position are contiguous, and `groups` groups of
// Cg = channels / groups neighbouring channels share a mean and a deviation over M = positions * Cg values:
//
//   h = (x - mean) * rstd      z = h * gamma + beta      out = act(z)
//   dz = out_grad * act'(z)    gamma_grad = sum dz * h   beta_grad = sum dz     (over samples and positions)
//   x_grad = rstd * (dz * gamma - mean_M(dz * gamma) - h * mean_M(dz * gamma * h))
//
// Both directions move every element of their operands once and compute a dozen or two operations on it, so
// they are bound by memory, and what counts is how often x is read.  A group's values are scattered (Cg
// neighbours out of every position), so a workgroup takes whole rows of a tile of neighbouring groups (which tile, and
// how the rows are dealt out: group_norm_plan.hpp).
//
// Statistics are held in f32 and never as a difference of large sums: a mean, and the sum of squared
// distances from it (merged as count, mean and that sum), in f64 where the parts of a group are joined.
// In the gradient h and z are each rounded as written (no fused multiply-add), so that the branch of an activation at
// z = 0 is the one that 32-bit arithmetic takes anywhere else.
#include <algorithm>
#include <cmath>

#include "group_norm_plan.hpp"
#include "op_device.hpp"
#include "runtime.hpp"

namespace custos_hip {

namespace {

using namespace group_norm;

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// n / d.by
__device__ __forceinline__ unsigned int divide(const Divisor& d, unsigned int n) {
    if (d.by == 1) return n;
    const unsigned int q = __umulhi(n, d.magic);  // (at most one too small)
    return n - q * d.by >= d.by ? q + 1 : q;
}

// e / per_group for e * per_group < 2^32 (0: per_group is 1).
__device__ __forceinline__ unsigned int group_of(unsigned int e, unsigned int magic) {
    return magic ? __umulhi(e, magic) : e;
}

// gamma or beta of V neighbouring channels, with one branch and wide loads.
template <class T, int V>
__device__ __forceinline__ void params(const void* p, int f32, unsigned int first, float none, float (&out)[V]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; j++) out[j] = none;
    } else if (f32) {
        constexpr int W = V >= 4 ? 4 : 1;
#pragma unroll
        for (int j = 0; j < V; j += W) {
            const Pack<float, W> v = load_pack<false, float, W>(static_cast<const float*>(p) + first + j);
#pragma unroll
            for (int k = 0; k < W; k++) out[j + k] = v.v[k];
        }
    } else {
        const Pack<T, V> v = load_pack<false, T, V>(static_cast<const T*>(p) + first);
#pragma unroll
        for (int j = 0; j < V; j++) out[j] = to_f32(v.v[j]);
    }
}

// Roundings may leave a sum of squares just below zero; a NaN stays one.
template <class F>
__device__ __forceinline__ F not_negative(F v) {
    return v < F(0) ? F(0) : v;
}

// exp(-z) through the hardware exp2: relative error below |z| 2^-24 + 1 ulp.
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
template <int ACT>
__device__ __forceinline__ float act(float z) {
    if (ACT == kRelu) return z < 0.0f ? 0.0f : z;
    if (ACT == kSilu) return z * sigmoid(z);
    if (ACT == kGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if (ACT == kRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == kSilu) {
        const float s = sigmoid(z);
        return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
    }
    if (ACT == kGelu)
        return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * (0.39894228f * __builtin_amdgcn_exp2f(z * z * -0.72134752f));
    return 1.0f;
}
// Which part of the data a thread of a tile works on: a vector of V channels, the same for all its rows.
// The last vector of a row of W channels starts at W - V; its first `dup` channels are also the vector
// before it's: they are not summed here, and stored by both with the same value (where that would not do, rows are
// worked on channel by channel: narrow_values).
struct Column {
    unsigned int width;   // channels of the tile
    unsigned int vecs;    // vectors per row
    unsigned int first;   // of the vector's channels, within the tile
    int dup;
};
template <int V>
__device__ __forceinline__ Column column_of(const GroupNormArgs& a, unsigned int col) {
    Column c;
    c.width = a.tile_groups * a.per_group;
    c.vecs = (c.width + V - 1) / V;
    c.first = col * V;
    c.dup = 0;
    if (c.first + V > c.width && col < c.vecs) {
        c.dup = static_cast<int>(c.first + V - c.width);
        c.first = c.width - V;
    }
    return c;
}

// x as the kernels read it: V elements of T, or of an 8-bit checkpoint.
template <class T, int V, bool SAVED>
struct Source {
    Bits<T, V> p;
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const GroupNormArgs& a, u64 row, unsigned int channel) {
        p.template load<STREAM>(static_cast<const T*>(a.x) + row * a.x_pitch + channel);
    }
    __device__ __forceinline__ void zero() { p.zero(); }
    __device__ __forceinline__ void forget_values() { p.forget_values(); }
    __device__ __forceinline__ float value(int j) const { return to_f32(p.pack().v[j]); }
};
template <class T, int V>
struct Source<T, V, true> {
    Bits<signed char, V> c;
    float low, high;  // the vector may end in the next block of 128
    int in_low;
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const GroupNormArgs& a, u64 row, unsigned int channel) {
        const u64 i = row * a.channels + channel;
        c.template load<STREAM>(a.codes + i);
        in_low = 128 - static_cast<int>(i & 127);
        low = a.scales[i >> 7];
        high = in_low < V ? a.scales[(i >> 7) + 1] : low;
    }
    __device__ __forceinline__ void zero() {
        c.zero();
        low = high = 0.0f;
        in_low = V;
    }
    __device__ __forceinline__ void forget_values() { c.forget_values(); }
    __device__ __forceinline__ float value(int j) const {
        const signed char code = c.pack().v[j];
        const float v = static_cast<float>(code) * (j < in_low ? low : high);
        return code == -128 ? __builtin_nanf("") : v;
    }
};

// How many values every channel of row `r` of a workgroup's threads stands for: `rounds`, one less from row `whole` on.
struct RowCounts {
    float rounds;
    unsigned int whole;
    __device__ __forceinline__ float of(unsigned int r) const { return r < whole ? rounds : rounds - 1.0f; }
};

// Mean and sum of squared distances of every group of a tile, from those of `step` x `width` channels (`table`):
// in f64, about the first entry's mean, so that no large numbers cancel.  All threads of the workgroup call it;
// result for group g in out[g], to be read after the return.
template <int THREADS>
__device__ __forceinline__ void merge_groups(const GroupNormArgs& a, const float2* table, const RowCounts& counts, float total_inverse, float2* out) {
    constexpr unsigned int kWaves = THREADS / 64;
    __shared__ double wave_sums[kWaves][2];
    const unsigned int t = threadIdx.x, width = a.tile_groups * a.per_group, entries = a.step * a.per_group;
    const bool shared = a.tile_groups < kWaves;  // several wavefronts per group, else several groups per wavefront
    unsigned int per = kWaves, lanes = 64;
    if (shared) per = a.waves_per_group;
    else
        while (lanes > 1 && lanes * a.tile_groups > static_cast<unsigned int>(THREADS)) lanes /= 2;
    __syncthreads();
    for (unsigned int base = 0; base < a.tile_groups; base += THREADS / lanes) {
        const unsigned int wave = t / 64, g = shared ? group_of(wave, a.waves_magic) : base + t / lanes;
        const unsigned int begin = shared ? (wave - g * per) * 64 + t % 64 : t % lanes, by = shared ? per * 64 : lanes;
        double first = 0.0, second = 0.0;
        float about = 0.0f;
        if (g < a.tile_groups) {
            about = table[g * a.per_group].x;
            for (unsigned int e = begin; e < entries; e += by) {
                const unsigned int r = group_of(e, a.per_group_magic);
                const float2 v = table[r * width + g * a.per_group + (e - r * a.per_group)];
                const double count = counts.of(r), d = v.x - about;
                first += count * d;
                second += v.y + count * d * d;
            }
        }
        for (unsigned int half = lanes / 2; half > 0; half /= 2) {
            first += __shfl_xor(first, half, 64);
            second += __shfl_xor(second, half, 64);
        }
        if (shared) {
            if (t % 64 == 0) wave_sums[wave][0] = first, wave_sums[wave][1] = second;
            __syncthreads();
            first = second = 0.0;
            if (t < a.tile_groups) {
                about = table[t * a.per_group].x;
                for (unsigned int i = 0; i < per; i++) first += wave_sums[t * per + i][0], second += wave_sums[t * per + i][1];
            }
        }
        const unsigned int mine = shared ? t : g;
        if (mine < a.tile_groups && (shared || t % lanes == 0)) {
            const double mean = first * total_inverse;
            out[mine] = make_float2(static_cast<float>(about + mean), static_cast<float>(not_negative(second - first * mean)));
        }
        if (shared) break;
    }
    __syncthreads();
}

// Sum over the workgroup, in every thread.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* wave_sums) {
    v = lanes_sum(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) wave_sums[threadIdx.x / 64] = v;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) total += wave_sums[w];
    return total;
}

template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v, double* wave_sums) {
    v = lanes_sum_f64(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) wave_sums[threadIdx.x / 64] = v;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) total += wave_sums[w];
    return total;
}

// The rows of a tile that one workgroup of a streaming kernel works on, and its threads' shares.  The workgroups of a
// sample take turns, `step` rows at a time, so that those that run together read neighbouring memory (each on a
// stretch of its own, at equal distances, they would meet in the same memory channels).
template <int V>
struct Stream {
    unsigned int n, part, tile, c0, vecs, step, r0, col0;
    u64 first, stride, rows;  // the thread's first row (of all samples), from row to row, and how many rows it has
    bool one_column;          // else a thread has several columns and every row
    __device__ __forceinline__ Stream(const GroupNormArgs& a, const Splits& of, unsigned int index) {
        const unsigned int t = threadIdx.x;
        const unsigned int block = divide(a.by_tiles, index);
        tile = index - block * a.tiles;
        const unsigned int sample = divide(of.by_count, block), split = block - sample * of.count;
        n = sample;
        part = block;
        vecs = a.vecs;
        one_column = vecs <= kBlock;
        step = a.step;
        r0 = one_column ? group_of(t, a.vecs_magic) : 0;
        col0 = one_column ? t - r0 * vecs : t;
        stride = static_cast<u64>(of.count) * step;
        const u64 p = static_cast<u64>(split) * step + r0;
        first = static_cast<u64>(n) * a.positions + p;
        rows = of.rounds + (split < of.longer ? 1 : 0);
        if (r0 >= step) rows = 0;
        else if (rows > 0 && p + (rows - 1) * stride >= a.positions) rows--;
        c0 = tile * a.tile_groups * a.per_group;
    }
    __device__ __forceinline__ bool active() const { return r0 < step; }
};

// Positions of part `split` of a sample.
__device__ __forceinline__ u64 part_rows(const GroupNormArgs& a, unsigned int split) {
    return (a.parts.rounds + (split < a.parts.longer ? 1 : 0)) * a.part_step - (split == a.last_part ? a.missing_rows : 0);
}

// Workgroups are dealt to the eight XCDs in turn, each with an L2 of its own.  This order gives an XCD neighbouring
// tiles, which share cache lines where a tile's rows are no whole lines.
__device__ __forceinline__ unsigned int by_xcd(unsigned int block, unsigned int blocks) {
    return blocks % 8 == 0 ? block % 8 * (blocks / 8) + block / 8 : block;
}

// ---- forward, a tile in registers: one launch, x read once ----

template <class T, int V, int HELD, int THREADS, int ACT>
__global__ void __launch_bounds__(THREADS) custos_group_norm_tile(const GroupNormArgs a) {
    __shared__ float2 table[THREADS * V];
    __shared__ float2 stats[kMaxTileGroups];
    const unsigned int t = threadIdx.x;
    const unsigned int index = by_xcd(blockIdx.x, gridDim.x), n = divide(a.by_tiles, index), tile = index - n * a.tiles;
    const unsigned int step = a.step;  // rows at a time
    const unsigned int r0 = group_of(t, a.vecs_magic);
    const Column c = column_of<V>(a, t - r0 * a.vecs);
    const bool active = r0 < step;
    const unsigned int c0 = tile * a.tile_groups * a.per_group, positions = static_cast<unsigned int>(a.positions);
    const T* x = static_cast<const T*>(a.x) + (static_cast<u64>(n) * a.positions + r0) * a.x_pitch + c0 + c.first;
    const unsigned int rounds = active && r0 < positions ? static_cast<unsigned int>(a.parts.rounds) - (r0 + (a.parts.rounds - 1) * step >= positions ? 1 : 0) : 0;
    Bits<T, V> held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (static_cast<unsigned int>(i) < rounds) held[i].load(x + static_cast<u64>(i) * step * a.x_pitch);
    float scale[V], shift[V];  // of the channels: gamma and beta until the statistics are there
    params<T, V>(a.gamma, a.param_f32, c0 + c.first, 1.0f, scale);
    params<T, V>(a.beta, a.param_f32, c0 + c.first, 0.0f, shift);
    // of the thread's channels: mean, then squared distances from it
    {
        float mean[V], m2[V];
#pragma unroll
        for (int j = 0; j < V; j++) mean[j] = m2[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            if (static_cast<unsigned int>(i) >= rounds) continue;
            const Pack<T, V> p = held[i].pack();
#pragma unroll
            for (int j = 0; j < V; j++) mean[j] += to_f32(p.v[j]);
            held[i].forget_values();
        }
        const float inverse = rounds > 0 ? 1.0f / static_cast<float>(rounds) : 0.0f;
#pragma unroll
        for (int j = 0; j < V; j++) mean[j] *= inverse;
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            if (static_cast<unsigned int>(i) >= rounds) continue;
            const Pack<T, V> p = held[i].pack();
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = to_f32(p.v[j]) - mean[j];
                m2[j] = __builtin_fmaf(d, d, m2[j]);
            }
            held[i].forget_values();
        }
        if (active) {
            float2* row = table + r0 * c.width + c.first;
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j >= c.dup) row[j] = make_float2(mean[j], m2[j]);
        }
    }
    const float total = static_cast<float>(a.positions) * static_cast<float>(a.per_group), total_inverse = 1.0f / total;
    const RowCounts counts{static_cast<float>(a.parts.rounds), step - a.missing_rows};
    merge_groups<THREADS>(a, table, counts, total_inverse, stats);
    if (t < a.tile_groups) {
        const float2 s = make_float2(stats[t].x, 1.0f / sqrtf(stats[t].y * total_inverse + a.eps));
        stats[t] = s;
        reinterpret_cast<float2*>(a.stats)[static_cast<u64>(n) * a.groups + tile * a.tile_groups + t] = s;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; j++) {
        const float2 s = stats[group_of(c.first + j, a.per_group_magic)];
        scale[j] *= s.y;
        shift[j] = __builtin_fmaf(-s.x, scale[j], shift[j]);
    }
    T* out = static_cast<T*>(a.out) + (static_cast<u64>(n) * a.positions + r0) * a.out_pitch + c0 + c.first;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        if (static_cast<unsigned int>(i) >= rounds) continue;
        const Pack<T, V> p = held[i].pack();
        Pack<T, V> y;
#pragma unroll
        for (int j = 0; j < V; j++) y.v[j] = from_f32<T>(act<ACT>(__builtin_fmaf(to_f32(p.v[j]), scale[j], shift[j])));
        store_pack<false, T, V>(out + static_cast<u64>(i) * step * a.out_pitch, y);
    }
}

// ---- forward, streaming: parts of every group and their join, then the values ----

// Mean and sum of squared distances of every group over the rows of one part.  A thread sums distances from the first
// value it meets in each channel, and after 8, 16, 32 ... rows goes over to the mean so far: were the first value an
// outlier, n squares of its distance would have to cancel in the end, and leave n^1.5 * 2^-24 of one of them (a deviation
// wrong by 1 % from some thousand rows on).
template <class T, int V>
__global__ void __launch_bounds__(kBlock) custos_group_norm_parts(const GroupNormArgs a) {
    __shared__ float2 table[kBlock * V];
    __shared__ double wave_sums[kBlock / 64];
    __shared__ float2 group[kMaxStreamGroups];
    const unsigned int t = threadIdx.x;
    const Stream<V> w(a, a.parts, blockIdx.x);
    float2* out = reinterpret_cast<float2*>(a.group_parts) + static_cast<u64>(w.part) * a.groups + w.tile * a.tile_groups;
    const float rows = static_cast<float>(w.rows);
    // One group per tile: sums over all columns of the thread, in f64 and about a value of the group that all threads of
    // the workgroup read, so that no large numbers cancel (as merge_groups has it for tiles of several).
    float base = 0.0f;
    if (a.tile_groups == 1) {
        Source<T, 1, false> x;
        x.load(a, w.first - w.r0, w.c0);
        base = x.value(0);
    }
    double all = 0.0, all_squares = 0.0;
    const double per_row = w.rows > 0 ? 1.0 / static_cast<double>(w.rows) : 0.0;
    float mean[V], m2[V];
    Column c = column_of<V>(a, w.col0);
    for (unsigned int col = w.col0; col < w.vecs && w.active(); col += kBlock) {
        c = column_of<V>(a, col);
        const unsigned int channel = w.c0 + c.first;
        float shift[V], s[V], q[V];
#pragma unroll
        for (int j = 0; j < V; j++) shift[j] = s[j] = q[j] = mean[j] = m2[j] = 0.0f;
        if (w.rows > 0) {
            Source<T, V, false> x;
            x.load(a, w.first, channel);
#pragma unroll
            for (int j = 0; j < V; j++) shift[j] = x.value(j);
        }
        auto add = [&](const Source<T, V, false>& x) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = x.value(j) - shift[j];
                s[j] += d;
                q[j] = __builtin_fmaf(d, d, q[j]);
            }
        };
        // distances from `to` in the place of those from shift: both sums follow, whatever the rounding of `to`
        auto go_over = [&](float n) {
            const float per = 1.0f / n;
#pragma unroll
            for (int j = 0; j < V; j++) {
                float to = __builtin_fmaf(s[j], per, shift[j]);
                if (!(fabsf(to) < __builtin_inff())) to = shift[j];  // (the group's results are NaN)
                const float moved = to - shift[j], left = __builtin_fmaf(-n, moved, s[j]);
                q[j] = not_negative(__builtin_fmaf(-moved, s[j] + left, q[j]));
                s[j] = left;
                shift[j] = to;
            }
        };
        constexpr int kAhead = kAheadForward;
        u64 i = 0, next = 2 * kAhead;
        for (; i + kAhead <= w.rows; i += kAhead) {
            Source<T, V, false> x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) x[u].load(a, w.first + (i + u) * w.stride, channel);
            if (i == next) {
                go_over(static_cast<float>(i));
                next *= 2;
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) add(x[u]);
        }
        for (; i < w.rows; i++) {
            Source<T, V, false> x;
            x.load(a, w.first + i * w.stride, channel);
            add(x);
        }
        if (w.rows > 0) {
            const float per = 1.0f / rows;
#pragma unroll
            for (int j = 0; j < V; j++) {
                mean[j] = __builtin_fmaf(s[j], per, shift[j]);
                m2[j] = not_negative(q[j] - s[j] * (s[j] * per));
            }
        }
        if (a.tile_groups == 1 && w.rows > 0) {
            double d1 = 0.0, d2 = 0.0;
            float squares = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const bool mine = j >= c.dup;
                const double d = mine ? __builtin_fma(s[j], per_row, static_cast<double>(shift[j]) - base) : 0.0;
                d1 += d;
                d2 = __builtin_fma(d, d, d2);
                squares += mine ? m2[j] : 0.0f;
            }
            all = __builtin_fma(rows, d1, all);
            all_squares = __builtin_fma(rows, d2, all_squares + squares);
        }
    }
    const unsigned int split = w.part - w.n * a.parts.count;
    const float total_inverse = 1.0f / (static_cast<float>(part_rows(a, split)) * static_cast<float>(a.per_group));
    if (a.tile_groups == 1) {
        all = block_sum_f64<kBlock>(all, wave_sums);
        all_squares = block_sum_f64<kBlock>(all_squares, wave_sums);
        const double m = all / (static_cast<double>(part_rows(a, split)) * a.per_group);
        if (t == 0) *out = make_float2(static_cast<float>(base + m), static_cast<float>(not_negative(all_squares - all * m)));
        return;
    }
    if (w.active()) {
        float2* row = table + w.r0 * c.width + c.first;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j >= c.dup) row[j] = make_float2(mean[j], m2[j]);
    }
    const RowCounts counts{static_cast<float>(a.parts.rounds + (split < a.parts.longer ? 1 : 0)), w.step - (split == a.last_part ? a.missing_rows : 0)};
    merge_groups<kBlock>(a, table, counts, total_inverse, group);
    for (unsigned int g = t; g < a.tile_groups; g += kBlock) out[g] = group[g];
}

// The parts of the tile's groups joined, in f64 and in a fixed order.  Every workgroup of the second pass does it for
// itself: at most 32 KiB, from the L2, against a launch of its own (4 to 5 us), or a last workgroup of the first
// pass that joins for all (the fences that needs between the L2s of the chip took 100 us of a pass of 80).
// `of(group, a, b)` receives each group's mean and deviation (FORWARD), or the two means of the gradient.
template <bool FORWARD, class F>
__device__ __forceinline__ void join_parts(const GroupNormArgs& a, unsigned int n, unsigned int tile, F of) {
    __shared__ double sums[2][kBlock];
    const unsigned int t = threadIdx.x;
    unsigned int lanes = 1;
    while (lanes * 2 * a.tile_groups <= static_cast<unsigned int>(kBlock)) lanes *= 2;
    const unsigned int lane = t / a.tile_groups, g = t - lane * a.tile_groups;
    const float2* part = reinterpret_cast<const float2*>(a.group_parts) + static_cast<u64>(n) * a.parts.count * a.groups + tile * a.tile_groups + g;
    double first = 0.0, second = 0.0;
    // means are taken from that of part 0, which is near all of them
    const double base = FORWARD ? part[0].x : 0.0;
    if (lane < lanes)
        for (unsigned int s = lane; s < a.parts.count; s += lanes) {
            const float2 v = part[static_cast<u64>(s) * a.groups];
            if (FORWARD) {
                const double count = static_cast<double>(part_rows(a, s)) * a.per_group, d = v.x - base;
                first += count * d;
                second += v.y + count * d * d;
            } else {
                first += v.x;
                second += v.y;
            }
        }
    sums[0][t] = first;
    sums[1][t] = second;
    for (unsigned int half = lanes / 2; half > 0; half /= 2) {
        __syncthreads();
        if (t < half * a.tile_groups) {
            sums[0][t] += sums[0][t + half * a.tile_groups];
            sums[1][t] += sums[1][t + half * a.tile_groups];
        }
    }
    if (t < a.tile_groups) {  // (its own sums)
        first = sums[0][t] * a.total_inverse;
        second = sums[1][t] * a.total_inverse;
        if (FORWARD) of(t, static_cast<float>(base + first), 1.0f / sqrtf(static_cast<float>(not_negative(second - first * first)) + a.eps));
        else of(t, static_cast<float>(first), static_cast<float>(second));
    }
    __syncthreads();
}

template <class T, int V, int ACT, bool STREAM>
__global__ void __launch_bounds__(kBlock) custos_group_norm_values(const GroupNormArgs a) {
    const Stream<V> w(a, a.values, a.blocks - 1 - blockIdx.x);  // (backwards: what the first pass read last is in the caches)
    __shared__ float2 stats[kMaxStreamGroups];
    float2* written = reinterpret_cast<float2*>(a.stats) + static_cast<u64>(w.n) * a.groups + w.tile * a.tile_groups;
    const bool writes = w.part == w.n * a.values.count;  // (one of the sample's workgroups writes the statistics down)
    join_parts<true>(a, w.n, w.tile, [&](unsigned int g, float mean, float rstd) {
        stats[g] = make_float2(mean, rstd);
        if (writes) written[g] = stats[g];
    });
    if (w.rows == 0) return;
    for (unsigned int col = w.col0; col < w.vecs; col += kBlock) {
        const Column c = column_of<V>(a, col);
        float scale[V], shift[V];
        params<T, V>(a.gamma, a.param_f32, w.c0 + c.first, 1.0f, scale);
        params<T, V>(a.beta, a.param_f32, w.c0 + c.first, 0.0f, shift);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const unsigned int g = a.tile_groups == 1 ? 0 : group_of(c.first + j, a.per_group_magic);
            const float2 mean_rstd = stats[g];
            scale[j] *= mean_rstd.y;
            shift[j] = __builtin_fmaf(-mean_rstd.x, scale[j], shift[j]);
        }
        T* out = static_cast<T*>(a.out) + w.c0 + c.first;
        {
            auto value = [&](const Source<T, V, false>& x) {
                Pack<T, V> y;
#pragma unroll
                for (int j = 0; j < V; j++)
                    y.v[j] = from_f32<T>(act<ACT>(__builtin_fmaf(x.value(j), scale[j], shift[j])));
                return y;
            };
            constexpr int kAhead = kAheadForward;
            u64 i = 0;
            for (; i + kAhead <= w.rows; i += kAhead) {
                Source<T, V, false> x[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) x[u].template load<STREAM>(a, w.first + (i + u) * w.stride, w.c0 + c.first);
#pragma unroll
                for (int u = 0; u < kAhead; u++) store_pack<STREAM, T, V>(out + (w.first + (i + u) * w.stride) * a.out_pitch, value(x[u]));
            }
            for (; i < w.rows; i++) {
                Source<T, V, false> x;
                x.template load<STREAM>(a, w.first + i * w.stride, w.c0 + c.first);
                store_pack<STREAM, T, V>(out + (w.first + i * w.stride) * a.out_pitch, value(x));
            }
        }
    }
}

// ---- backward ----

// What a thread needs of its column's channels.
template <class T, int V>
struct ChannelParams {
    float mean[V], rstd[V], gamma[V], beta[V];
    __device__ __forceinline__ void load(const GroupNormArgs& a, unsigned int n, unsigned int tile, const Column& c) {
        const unsigned int c0 = tile * a.tile_groups * a.per_group;
        const float2* stats = reinterpret_cast<const float2*>(a.stats) + static_cast<u64>(n) * a.groups + tile * a.tile_groups;
        params<T, V>(a.gamma, a.param_f32, c0 + c.first, 1.0f, gamma);
        params<T, V>(a.beta, a.param_f32, c0 + c.first, 0.0f, beta);
        if (a.whole_groups) {  // (the vector's channels are one group's)
            const float2 s = stats[a.tile_groups == 1 ? 0 : group_of(c.first, a.per_group_magic)];
#pragma unroll
            for (int j = 0; j < V; j++) mean[j] = s.x, rstd[j] = s.y;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float2 s = stats[group_of(c.first + j, a.per_group_magic)];
                mean[j] = s.x;
                rstd[j] = s.y;
            }
        }
    }
};

// dz and h of element j of a column.
template <int ACT, class T, int V>
__device__ __forceinline__ float dz_of(const ChannelParams<T, V>& k, int j, float x, float out_grad, float* h) {
    *h = (x - k.mean[j]) * k.rstd[j];
    const float z = *h * k.gamma[j] + k.beta[j];
    return out_grad * act_grad<ACT>(z);
}

// x_grad = rstd * (dz * gamma - mean_dh - h * mean_dhh), the rstd multiplied in beforehand.
template <class T, int V>
struct GradientOf {
    float on_dz[V], on_h[V], constant[V];
    template <class F>
    __device__ __forceinline__ GradientOf(const ChannelParams<T, V>& k, F means_of) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            float dh, dhh;
            means_of(j, &dh, &dhh);
            on_dz[j] = k.rstd[j] * k.gamma[j];
            on_h[j] = -k.rstd[j] * dhh;
            constant[j] = -k.rstd[j] * dh;
        }
    }
    __device__ __forceinline__ float of(int j, float dz, float h) const {
        return __builtin_fmaf(dz, on_dz[j], __builtin_fmaf(h, on_h[j], constant[j]));
    }
};

template <bool STREAM, class T, int V>
__device__ __forceinline__ void store_grad(const GroupNormArgs& a, T* p, float (&g)[V]) {
    Pack<T, V> y;
    if (a.accumulate) {
        const Pack<T, V> was = load_pack<false, T, V>(p);
#pragma unroll
        for (int j = 0; j < V; j++) g[j] += to_f32(was.v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; j++) y.v[j] = from_f32<T>(g[j]);
    store_pack<STREAM, T, V>(p, y);
}

// From a thread's sums s1 (dz) and s2 (dz * h) of its column: those of the channels over the rows of the workgroup,
// to `channel` (`adds`: to what the same thread put there), and from there, times gamma, those of the groups, to sums_of.
template <int V, int THREADS>
__device__ __forceinline__ void channel_and_group_sums(const GroupNormArgs& a, const Column& c, unsigned int r0, unsigned int step,
                                                       const float (&s1)[V], const float (&s2)[V], const float (&gamma_of)[V], float2* table, float* gammas,
                                                       float* channel, bool adds, float2* sums_of) {
    const unsigned int t = threadIdx.x;
    if (r0 == 0) {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j >= c.dup) gammas[c.first + j] = gamma_of[j];
    }
    if (r0 < step) {
        float2* row = table + r0 * c.width + c.first;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j >= c.dup) row[j] = make_float2(s1[j], s2[j]);
    }
    __syncthreads();
    // (a power of two of neighbouring lanes for each channel, then for each group)
    unsigned int lanes = 1;
    while (lanes < 64 && lanes * 2 * c.width <= static_cast<unsigned int>(THREADS) && lanes < step) lanes *= 2;
    for (unsigned int base = 0; base < c.width; base += THREADS / lanes) {
        const unsigned int ch = base + t / lanes;
        float x = 0.0f, y = 0.0f;
        if (ch < c.width)
            for (unsigned int r = t % lanes; r < step; r += lanes) {
                const float2 v = table[r * c.width + ch];
                x += v.x;
                y += v.y;
            }
        for (unsigned int half = lanes / 2; half > 0; half /= 2) x += __shfl_xor(x, half, 64), y += __shfl_xor(y, half, 64);
        if (ch < c.width && t % lanes == 0) {
            channel[ch] = adds ? channel[ch] + x : x;
            channel[a.channels + ch] = adds ? channel[a.channels + ch] + y : y;
            const float gamma = gammas[ch];
            table[ch] = make_float2(x * gamma, y * gamma);  // (only these lanes read column ch, and they have)
        }
    }
    __syncthreads();
    lanes = 1;
    while (lanes < 64 && lanes * 2 * a.tile_groups <= static_cast<unsigned int>(THREADS) && lanes < a.per_group) lanes *= 2;
    for (unsigned int base = 0; base < a.tile_groups; base += THREADS / lanes) {
        const unsigned int g = base + t / lanes;
        float x = 0.0f, y = 0.0f;
        if (g < a.tile_groups)
            for (unsigned int i = t % lanes; i < a.per_group; i += lanes) {
                const float2 v = table[g * a.per_group + i];
                x += v.x;
                y += v.y;
            }
        for (unsigned int half = lanes / 2; half > 0; half /= 2) x += __shfl_xor(x, half, 64), y += __shfl_xor(y, half, 64);
        if (g < a.tile_groups && t % lanes == 0) sums_of[g] = make_float2(x, y);
    }
    __syncthreads();
}

// gamma_grad and beta_grad of 16 channels, by one workgroup: the sums of all parts of all samples, in a fixed order.
constexpr int kParamChannels = 16;
__device__ __forceinline__ void param_grads(const GroupNormArgs& a, unsigned int block, double* sums) {
    const unsigned int t = threadIdx.x, which = t / kParamChannels % 2, lane = t / (2 * kParamChannels);
    constexpr unsigned int kLanes = kBlock / (2 * kParamChannels);
    const unsigned int ch = block * kParamChannels + t % kParamChannels;
    double s = 0.0;
    if (ch < a.channels)
#pragma unroll 4
        for (unsigned int row = lane; row < a.channel_rows; row += kLanes)
            s += a.channel_parts[(static_cast<u64>(row) * 2 + which) * a.channels + ch];
    sums[t] = s;
    __syncthreads();
    if (lane > 0 || ch >= a.channels) return;
    for (unsigned int l = 1; l < kLanes; l++) s += sums[l * 2 * kParamChannels + t];
    float* out = which ? a.gamma_grad : a.beta_grad;
    if (out) out[ch] = static_cast<float>(a.accumulate ? out[ch] + s : s);
}

__global__ void __launch_bounds__(kBlock) custos_group_norm_param_grads(const GroupNormArgs a) {
    __shared__ double sums[kBlock];
    param_grads(a, blockIdx.x, sums);
}

// A tile in registers: x and out_grad read once.  With more samples than the chip holds workgroups for, each takes
// several, `channel_rows` apart, so that the work area and what is added up behind stay small.  (Nothing in shared
// memory is written again before a barrier that follows its last read.)
template <class T, int V, int HELD, int THREADS, bool SAVED, int ACT>
__global__ void __launch_bounds__(THREADS) custos_group_norm_grad_tile(const GroupNormArgs a) {
    __shared__ float2 table[THREADS * V];
    __shared__ float gammas[THREADS * V];
    __shared__ float2 sums_of[kMaxTileGroups];
    const unsigned int t = threadIdx.x;
    const unsigned int index = by_xcd(blockIdx.x, gridDim.x), sample0 = divide(a.by_tiles, index), tile = index - sample0 * a.tiles;
    const unsigned int vecs = a.vecs, step = a.step;
    const unsigned int r0 = group_of(t, a.vecs_magic);
    const Column c = column_of<V>(a, t - r0 * vecs);
    const bool active = r0 < step;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    for (unsigned int n = sample0; n < a.samples; n += a.channel_rows) {
        const u64 row0 = static_cast<u64>(n) * a.positions;
        const T* out_grad = static_cast<const T*>(a.out_grad) + row0 * a.grad_pitch + c0 + c.first;
        Source<T, V, SAVED> held[HELD];
        Bits<T, V> grad[HELD];
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const u64 p = r0 + static_cast<u64>(i) * step;
            if (active && p < a.positions) {
                held[i].load(a, row0 + p, c0 + c.first);
                grad[i].load(out_grad + p * a.grad_pitch);
            } else {
                held[i].zero();
                grad[i].zero();
            }
        }
        ChannelParams<T, V> k;
        k.load(a, n, tile, c);
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.0f;
        {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                if (r0 + static_cast<u64>(i) * step >= a.positions) break;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<ACT>(k, j, held[i].value(j), to_f32(grad[i].pack().v[j]), &h);
                    s1[j] += dz;
                    s2[j] = __builtin_fmaf(dz, h, s2[j]);
                }
                held[i].forget_values();
                grad[i].forget_values();
            }
        }
        channel_and_group_sums<V, THREADS>(a, c, r0, step, s1, s2, k.gamma, table, gammas, a.channel_parts + static_cast<u64>(sample0) * 2 * a.channels + c0, n != sample0, sums_of);
        if (!a.out || !active) continue;
        const float count = static_cast<float>(a.positions) * static_cast<float>(a.per_group);
        const GradientOf<T, V> gradient(k, [&](int j, float* dh, float* dhh) {
            const unsigned int g = group_of(c.first + j, a.per_group_magic);
            const float2 both = sums_of[g];
            *dh = both.x / count;
            *dhh = both.y / count;
        });
        T* out = static_cast<T*>(a.out) + row0 * a.out_pitch + c0 + c.first;
        {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const u64 p = r0 + static_cast<u64>(i) * step;
                if (p >= a.positions) break;
                float g[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<ACT>(k, j, held[i].value(j), to_f32(grad[i].pack().v[j]), &h);
                    g[j] = gradient.of(j, dz, h);
                }
                store_grad<false, T, V>(a, out + p * a.out_pitch, g);
            }
        }
    }
}

// Rows of x and out_grad, `kAhead` of them loaded before they are used.
template <class T, int V, bool SAVED, bool STREAM, class F>
__device__ __forceinline__ void for_rows(const GroupNormArgs& a, const Stream<V>& w, unsigned int channel, F f) {
    const T* out_grad = static_cast<const T*>(a.out_grad) + channel;
    constexpr int kAhead = kAheadBackward;
    u64 i = 0;
    for (; i + kAhead <= w.rows; i += kAhead) {
        Source<T, V, SAVED> x[kAhead];
        Bits<T, V> g[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const u64 row = w.first + (i + u) * w.stride;
            x[u].template load<STREAM>(a, row, channel);
            g[u].template load<STREAM>(out_grad + row * a.grad_pitch);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) f(w.first + (i + u) * w.stride, x[u], g[u].pack());
    }
    for (; i < w.rows; i++) {
        const u64 row = w.first + i * w.stride;
        Source<T, V, SAVED> x;
        Bits<T, V> g;
        x.template load<STREAM>(a, row, channel);
        g.template load<STREAM>(out_grad + row * a.grad_pitch);
        f(row, x, g.pack());
    }
}

// Sums of dz and dz * h over the rows of one part: per channel, and times gamma per group.
template <class T, int V, bool SAVED, int ACT>
__global__ void __launch_bounds__(kBlock) custos_group_norm_grad_parts(const GroupNormArgs a) {
    __shared__ float2 table[kBlock * V];
    __shared__ float gammas[kBlock * V];
    __shared__ float2 sums_of[kMaxStreamGroups];
    __shared__ float wave_sums[kBlock / 64];
    const unsigned int t = threadIdx.x;
    const Stream<V> w(a, a.parts, blockIdx.x);
    float* channel = a.channel_parts + static_cast<u64>(w.part) * 2 * a.channels + w.c0;
    float* group = a.group_parts + (static_cast<u64>(w.part) * a.groups + w.tile * a.tile_groups) * 2;
    float s1[V], s2[V], dh = 0.0f, dhh = 0.0f;
    ChannelParams<T, V> k;
#pragma unroll
    for (int j = 0; j < V; j++) s1[j] = s2[j] = k.gamma[j] = 0.0f;
    Column c = column_of<V>(a, w.col0);
    for (unsigned int col = w.col0; col < w.vecs && w.active(); col += kBlock) {
        c = column_of<V>(a, col);
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.0f;
        k.load(a, w.n, w.tile, c);
        {
            for_rows<T, V, SAVED, false>(a, w, w.c0 + c.first, [&](u64, const Source<T, V, SAVED>& x, const Pack<T, V>& g) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<ACT>(k, j, x.value(j), to_f32(g.v[j]), &h);
                    s1[j] += dz;
                    s2[j] = __builtin_fmaf(dz, h, s2[j]);
                }
            });
        }
        if (!w.one_column) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j >= c.dup) {
                    channel[c.first + j] = s1[j], channel[a.channels + c.first + j] = s2[j];
                    dh = __builtin_fmaf(s1[j], k.gamma[j], dh);
                    dhh = __builtin_fmaf(s2[j], k.gamma[j], dhh);
                }
        }
    }
    if (!w.one_column) {
        dh = block_sum<kBlock>(dh, wave_sums);
        dhh = block_sum<kBlock>(dhh, wave_sums);
        if (t == 0) group[0] = dh, group[1] = dhh;
        return;
    }
    channel_and_group_sums<V, kBlock>(a, c, w.r0, w.step, s1, s2, k.gamma, table, gammas, channel, false, sums_of);
    for (unsigned int g = t; g < a.tile_groups; g += kBlock) reinterpret_cast<float2*>(group)[g] = sums_of[g];
}

// x_grad, and by the workgroups behind the first `blocks` gamma_grad and beta_grad.
template <class T, int V, bool SAVED, int ACT, bool STREAM>
__global__ void __launch_bounds__(kBlock) custos_group_norm_grad_values(const GroupNormArgs a) {
    __shared__ double sums[kBlock];
    if (blockIdx.x >= a.blocks) {
        param_grads(a, blockIdx.x - a.blocks, sums);
        return;
    }
    const Stream<V> w(a, a.values, a.blocks - 1 - blockIdx.x);  // (backwards: what the first pass read last is in the caches)
    __shared__ float2 means[kMaxStreamGroups];
    join_parts<false>(a, w.n, w.tile, [&](unsigned int g, float dh, float dhh) { means[g] = make_float2(dh, dhh); });
    if (w.rows == 0) return;
    for (unsigned int col = w.col0; col < w.vecs; col += kBlock) {
        const Column c = column_of<V>(a, col);
        ChannelParams<T, V> k;
        k.load(a, w.n, w.tile, c);
        const GradientOf<T, V> gradient(k, [&](int j, float* dh, float* dhh) {
            const unsigned int g = a.tile_groups == 1 ? 0 : group_of(c.first + j, a.per_group_magic);
            const float2 both = means[g];
            *dh = both.x;
            *dhh = both.y;
        });
        T* out = static_cast<T*>(a.out) + w.c0 + c.first;
        {
            for_rows<T, V, SAVED, STREAM>(a, w, w.c0 + c.first, [&](u64 row, const Source<T, V, SAVED>& x, const Pack<T, V>& og) {
                float g[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<ACT>(k, j, x.value(j), to_f32(og.v[j]), &h);
                    g[j] = gradient.of(j, dz, h);
                }
                store_grad<STREAM, T, V>(a, out + row * a.out_pitch, g);
            });
        }
    }
}

// ---- host ----

int32_t check_desc(custos_hip_device* dev, const char* what, const custos_hip_group_norm_desc* d) {
    auto bad = [&](const char* why) { return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why); };
    if (!d) return bad("the description is null");
    if (d->dtype != CUSTOS_HIP_F32 && d->dtype != CUSTOS_HIP_F16 && d->dtype != CUSTOS_HIP_BF16) return bad("elements are f32, f16 or bf16");
    if (d->param_dtype != CUSTOS_HIP_F32 && d->param_dtype != d->dtype) return bad("gamma and beta are f32 or of the element type");
    if (d->activation < 0 || d->activation > CUSTOS_HIP_ACT_GELU) return bad("unknown activation");
    if (d->flags & ~CUSTOS_HIP_GRAD_OVERWRITE) return bad("unknown flag");
    if (d->channels == 0 || d->groups == 0 || d->channels % d->groups != 0) return bad("the channels divide into the groups");
    // (as the kernels hold it: a group of equal values divides by its root)
    if (!(d->eps > 0) || !std::isnormal(static_cast<float>(d->eps))) return bad("eps is positive, and a normal number in f32");
    if (d->channels >= (1ull << 30) || d->samples >= (1ull << 31) || d->positions >= (1ull << 40) ||
        static_cast<double>(d->samples) * static_cast<double>(d->positions) * static_cast<double>(d->channels) > 1e15)
        return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": the sizes are beyond any memory");
    return CUSTOS_HIP_OK;
}

// A plan outside what the kernels hold would write past their shared arrays.
int32_t check_plan(custos_hip_device* dev, const char* what, const Plan& plan) {
    if (fits(plan)) return CUSTOS_HIP_OK;
    return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": no kernel holds a tile of these sizes");
}

template <class K>
void* handle(K* kernel) {
    return reinterpret_cast<void*>(kernel);
}

struct Kernel {
    void* fn;
    const char* name;
};

// Kernels by plan, element type, activation, and whether x is a checkpoint.
template <class T, int ACT>
Kernel forward_tile(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_tile";
    const bool wide = p.vec > 1;
    if (!wide) {  // (rows of less than a vector, and rows that are no whole vectors in place)
        if (p.threads == 256) return {handle(custos_group_norm_tile<T, 1, 8, 256, ACT>), name};
        return {handle(custos_group_norm_tile<T, 1, 16, 1024, ACT>), name};
    }
    if (p.threads == 256) return {p.held == 4 ? handle(custos_group_norm_tile<T, V, 4, 256, ACT>) : handle(custos_group_norm_tile<T, V, 8, 256, ACT>), name};
    if (p.held == 4) return {handle(custos_group_norm_tile<T, V, 4, 1024, ACT>), name};
    return {p.held == 8 ? handle(custos_group_norm_tile<T, V, 8, 1024, ACT>) : handle(custos_group_norm_tile<T, V, 16, 1024, ACT>), name};
}
template <class T>
Kernel forward_parts(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_parts<T, V>) : handle(custos_group_norm_parts<T, 1>), "custos_group_norm_parts"};
}
template <class T, int ACT>
Kernel forward_values(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_values";
    if (p.vec == 1) return {handle(custos_group_norm_values<T, 1, ACT, false>), name};
    return {p.stream ? handle(custos_group_norm_values<T, V, ACT, true>) : handle(custos_group_norm_values<T, V, ACT, false>), name};
}
template <class T, int ACT, bool SAVED>
Kernel backward_tile(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_grad_tile";
    const bool wide = p.vec > 1;
    if (p.threads == 512)
        return {wide ? handle(custos_group_norm_grad_tile<T, V, 4, 512, SAVED, ACT>) : handle(custos_group_norm_grad_tile<T, 1, 4, 512, SAVED, ACT>), name};
    return {wide ? handle(custos_group_norm_grad_tile<T, V, 4, 256, SAVED, ACT>) : handle(custos_group_norm_grad_tile<T, 1, 4, 256, SAVED, ACT>), name};
}
template <class T, int ACT, bool SAVED>
Kernel backward_parts(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_grad_parts<T, V, SAVED, ACT>) : handle(custos_group_norm_grad_parts<T, 1, SAVED, ACT>),
            "custos_group_norm_grad_parts"};
}
template <class T, int ACT, bool SAVED>
Kernel backward_values(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_grad_values";
    if (p.vec == 1) return {handle(custos_group_norm_grad_values<T, 1, SAVED, ACT, false>), name};
    return {p.stream ? handle(custos_group_norm_grad_values<T, V, SAVED, ACT, true>) : handle(custos_group_norm_grad_values<T, V, SAVED, ACT, false>), name};
}

// `pick(element type, activation)`
template <class T, class F>
Kernel by_activation(int32_t activation, F pick) {
    switch (activation) {
        case CUSTOS_HIP_ACT_RELU: return pick(T(), std::integral_constant<int, kRelu>());
        case CUSTOS_HIP_ACT_SILU: return pick(T(), std::integral_constant<int, kSilu>());
        case CUSTOS_HIP_ACT_GELU: return pick(T(), std::integral_constant<int, kGelu>());
        default: return pick(T(), std::integral_constant<int, kNone>());
    }
}
template <class F>
Kernel kernel_for(const custos_hip_group_norm_desc& d, F pick) {
    if (d.dtype == CUSTOS_HIP_F32) return by_activation<float>(d.activation, pick);
    if (d.dtype == CUSTOS_HIP_F16) return by_activation<_Float16>(d.activation, pick);
    return by_activation<__bf16>(d.activation, pick);
}

int32_t launch(custos_hip_device* dev, const Kernel& k, u64 blocks, int threads, const GroupNormArgs& a, const Access* acc, size_t n_acc) {
    const OpArg arg{&a, sizeof a};
    OpLaunch op{};
    op.name = k.name;
    op.func = k.fn;
    op.grid = dim3(static_cast<unsigned int>(blocks));
    op.block = dim3(static_cast<unsigned int>(threads));
    op.args = &arg;
    op.n_args = 1;
    op.acc = acc;
    op.n_acc = n_acc;
    return launch_op(dev, op);
}

}  // namespace

}  // namespace custos_hip

using namespace custos_hip;

extern "C" {

int32_t custos_hip_group_norm(custos_hip_device* dev, const custos_hip_group_norm_desc* desc, uint64_t x, uint64_t x_pitch,
                              uint64_t gamma, uint64_t beta, uint64_t out, uint64_t out_pitch, uint64_t stats) {
    int32_t rc = check_desc(dev, "group norm", desc);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (desc->flags != 0) return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, "group norm: the forward pass takes no flags");
    if (desc->samples == 0 || desc->positions == 0) {
        REQUIRE_DEV(dev);
        return CUSTOS_HIP_OK;
    }
    const size_t es = elem_size(desc->dtype), ps = elem_size(desc->param_dtype);
    const u64 rows = desc->samples * desc->positions;
    Operand ops[5] = {{"out", out, rows, desc->channels * es, out_pitch * es, true, es, true},
                      {"stats", stats, 1, desc->samples * desc->groups * 8, 0, true, 4},
                      {"x", x, rows, desc->channels * es, x_pitch * es, false, es, true}};
    size_t n = 3;
    if (gamma) ops[n++] = {"gamma", gamma, 1, desc->channels * ps, 0, false, ps};
    if (beta) ops[n++] = {"beta", beta, 1, desc->channels * ps, 0, false, ps};
    rc = check_operands(dev, "group norm", ops, n);
    if (rc != CUSTOS_HIP_OK) return rc;

    Plan plan = forward_plan(*desc);
    rc = check_plan(dev, "group norm", plan);
    if (rc != CUSTOS_HIP_OK) return rc;
    GroupNormArgs& a = plan.a;
    a.x = reinterpret_cast<const void*>(x);
    a.gamma = reinterpret_cast<const void*>(gamma);
    a.beta = reinterpret_cast<const void*>(beta);
    a.out = reinterpret_cast<void*>(out);
    a.stats = reinterpret_cast<float*>(stats);
    a.x_pitch = x_pitch;
    a.out_pitch = out_pitch;
    a.param_f32 = desc->param_dtype == CUSTOS_HIP_F32;
    Access acc[6];
    for (size_t i = 0; i < n; i++) acc[i] = ops[i].access();
    const u64 parts = static_cast<u64>(a.samples) * a.parts.count, blocks = parts * a.tiles;
    rc = check_grid(dev, "group norm", plan.in_registers ? blocks : static_cast<u64>(a.samples) * a.tiles * std::max(a.parts.count, a.values.count), plan.threads);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    if (plan.in_registers)
        return launch(dev, kernel_for(*desc, [&](auto t, auto act) { return forward_tile<decltype(t), act.value>(plan); }), blocks, plan.threads, a, acc, n);

    const size_t part_bytes = parts * a.groups * 2 * sizeof(float);
    uint64_t area = 0;
    rc = operator_workspace(dev, part_bytes, &area);
    if (rc != CUSTOS_HIP_OK) return rc;
    a.group_parts = reinterpret_cast<float*>(area);
    const Access in_parts[2] = {ops[2].access(), {area, area + part_bytes, true}};
    acc[n] = {area, area + part_bytes, false};
    rc = launch(dev, kernel_for(*desc, [&](auto t, auto) { return forward_parts<decltype(t)>(plan); }), blocks, kBlock, a, in_parts, 2);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (out == x) narrow_values(&plan);
    a.blocks = static_cast<unsigned int>(static_cast<u64>(a.samples) * a.tiles * a.values.count);
    return launch(dev, kernel_for(*desc, [&](auto t, auto act) { return forward_values<decltype(t), act.value>(plan); }), a.blocks, kBlock, a, acc,
                  n + 1);
}

int32_t custos_hip_add_group_norm_grad(custos_hip_device* dev, const custos_hip_group_norm_desc* desc, uint64_t x, uint64_t x_pitch,
                                       uint64_t codes, uint64_t scales, uint64_t stats, uint64_t gamma, uint64_t beta,
                                       uint64_t out_grad, uint64_t out_grad_pitch, uint64_t x_grad, uint64_t x_grad_pitch,
                                       uint64_t gamma_grad, uint64_t beta_grad) {
    const char* what = "group norm gradient";
    int32_t rc = check_desc(dev, what, desc);
    if (rc != CUSTOS_HIP_OK) return rc;
    const bool saved = x == 0;
    if (saved ? !codes || !scales : codes || scales)
        return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": x is given either as values or as codes and scales");
    const bool overwrite = (desc->flags & CUSTOS_HIP_GRAD_OVERWRITE) != 0;
    const size_t es = elem_size(desc->dtype), ps = elem_size(desc->param_dtype);
    const u64 rows = desc->samples * desc->positions, total = rows * desc->channels;
    if (rows == 0) {
        REQUIRE_DEV(dev);
        if (overwrite && gamma_grad) rc = custos_hip_clear(dev, gamma_grad, desc->channels * 4);
        if (rc == CUSTOS_HIP_OK && overwrite && beta_grad) rc = custos_hip_clear(dev, beta_grad, desc->channels * 4);
        return rc;
    }
    Operand ops[9];
    size_t n = 0;
    if (x_grad) ops[n++] = {"x_grad", x_grad, rows, desc->channels * es, x_grad_pitch * es, true, es, overwrite};
    const size_t values_written = n;
    if (gamma_grad) ops[n++] = {"gamma_grad", gamma_grad, 1, desc->channels * 4, 0, true, 4};
    if (beta_grad) ops[n++] = {"beta_grad", beta_grad, 1, desc->channels * 4, 0, true, 4};
    const size_t first_read = n;
    ops[n++] = {"out_grad", out_grad, rows, desc->channels * es, out_grad_pitch * es, false, es, true};
    if (saved) {
        ops[n++] = {"codes", codes, 1, total, 0, false, 1};
        ops[n++] = {"scales", scales, 1, (total + 127) / 128 * 4, 0, false, 4};
    } else {
        ops[n++] = {"x", x, rows, desc->channels * es, x_pitch * es, false, es, true};
    }
    ops[n++] = {"stats", stats, 1, desc->samples * desc->groups * 8, 0, false, 4};
    if (gamma) ops[n++] = {"gamma", gamma, 1, desc->channels * ps, 0, false, ps};
    if (beta) ops[n++] = {"beta", beta, 1, desc->channels * ps, 0, false, ps};
    static_assert(sizeof ops / sizeof ops[0] >= 9, "three written, six read");
    rc = check_operands(dev, what, ops, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (first_read == 0) {  // no gradient is wanted
        REQUIRE_DEV(dev);
        return CUSTOS_HIP_OK;
    }

    Plan plan = gradient_plan(*desc, saved);
    rc = check_plan(dev, what, plan);
    if (rc != CUSTOS_HIP_OK) return rc;
    GroupNormArgs& a = plan.a;
    a.x = reinterpret_cast<const void*>(x);
    a.codes = reinterpret_cast<const signed char*>(codes);
    a.scales = reinterpret_cast<const float*>(scales);
    a.gamma = reinterpret_cast<const void*>(gamma);
    a.beta = reinterpret_cast<const void*>(beta);
    a.out_grad = reinterpret_cast<const void*>(out_grad);
    a.out = reinterpret_cast<void*>(x_grad);
    a.stats = reinterpret_cast<float*>(stats);
    a.x_pitch = x_pitch;
    a.grad_pitch = out_grad_pitch;
    a.out_pitch = x_grad_pitch;
    a.param_f32 = desc->param_dtype == CUSTOS_HIP_F32;
    a.accumulate = !overwrite;
    const u64 parts = static_cast<u64>(a.samples) * a.parts.count;
    a.channel_rows = static_cast<unsigned int>(parts);
    if (plan.in_registers) {
        const u64 together = std::max<u64>(1, kThreadsTogether / (static_cast<u64>(plan.threads) * a.tiles)), each = (parts + together - 1) / together;
        a.channel_rows = static_cast<unsigned int>((parts + each - 1) / each);
    }
    const u64 blocks = static_cast<u64>(a.channel_rows) * a.tiles;
    rc = check_grid(dev, what, plan.in_registers ? blocks : static_cast<u64>(a.samples) * a.tiles * std::max(a.parts.count, a.values.count) + a.channels, plan.threads);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    const size_t channel_bytes = static_cast<u64>(a.channel_rows) * 2 * a.channels * sizeof(float), part_bytes = plan.in_registers ? 0 : parts * a.groups * 2 * sizeof(float);
    const size_t area_bytes = channel_bytes + part_bytes;
    uint64_t area = 0;
    rc = operator_workspace(dev, area_bytes, &area);
    if (rc != CUSTOS_HIP_OK) return rc;
    a.group_parts = reinterpret_cast<float*>(area);
    a.channel_parts = reinterpret_cast<float*>(area + part_bytes);
    a.gamma_grad = reinterpret_cast<float*>(gamma_grad);
    a.beta_grad = reinterpret_cast<float*>(beta_grad);
    const Access area_written{area, area + area_bytes, true}, area_read{area, area + area_bytes, false};
    // what every launch reads, then what it writes
    Access acc[12];
    size_t n_read = 0;
    for (size_t i = first_read; i < n; i++) acc[n_read++] = ops[i].access();
    const u64 param_blocks = gamma_grad || beta_grad ? (a.channels + kParamChannels - 1) / kParamChannels : 0;
    Access in_params[3] = {area_read, {}, {}};
    size_t n_params = 1;
    for (size_t i = values_written; i < first_read; i++) in_params[n_params++] = ops[i].access();
    if (plan.in_registers || !x_grad) {
        size_t n_acc = n_read;
        if (plan.in_registers && x_grad) acc[n_acc++] = ops[0].access();
        acc[n_acc++] = area_written;
        rc = launch(dev, kernel_for(*desc, [&](auto t, auto act) {
                        using T = decltype(t);
                        constexpr int ACT = act.value;
                        if (plan.in_registers) return saved ? backward_tile<T, ACT, true>(plan) : backward_tile<T, ACT, false>(plan);
                        return saved ? backward_parts<T, ACT, true>(plan) : backward_parts<T, ACT, false>(plan);
                    }), blocks, plan.threads, a, acc, n_acc);
        if (rc != CUSTOS_HIP_OK || param_blocks == 0) return rc;
        return launch(dev, {handle(custos_group_norm_param_grads), "custos_group_norm_param_grads"}, param_blocks, kBlock, a, in_params, n_params);
    }
    acc[n_read] = area_written;
    rc = launch(dev, kernel_for(*desc, [&](auto t, auto act) { return saved ? backward_parts<decltype(t), act.value, true>(plan) : backward_parts<decltype(t), act.value, false>(plan); }),
                blocks, kBlock, a, acc, n_read + 1);
    if (rc != CUSTOS_HIP_OK) return rc;
    size_t n_acc = n_read;
    acc[n_acc++] = area_read;
    acc[n_acc++] = ops[0].access();
    for (size_t i = 1; i < n_params; i++) acc[n_acc++] = in_params[i];
    if (!overwrite || x_grad == x || x_grad == out_grad) narrow_values(&plan);
    a.blocks = static_cast<unsigned int>(static_cast<u64>(a.samples) * a.tiles * a.values.count);
    return launch(dev, kernel_for(*desc, [&](auto t, auto act) { return saved ? backward_values<decltype(t), act.value, true>(plan) : backward_values<decltype(t), act.value, false>(plan); }),
                  a.blocks + param_blocks, kBlock, a, acc, n_acc);
}

}  // extern "C"
