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
// neighbours out of every position), so a workgroup takes whole rows of a tile of neighbouring groups.
//
// Statistics are held in f32 and never as a difference of large sums: a mean, and the sum of squared
// distances from it (merged as count, mean and that sum), in f64 where the parts of a group are joined.
// h and z are each rounded as written (no fused multiply-add), so that the branch of an activation at
// z = 0 is the one that 32-bit arithmetic takes anywhere else.
#include <algorithm>
#include <cmath>

#include "op_device.hpp"
#include "runtime.hpp"

namespace custos_hip {

namespace {

constexpr int kBlock = 256;      // threads of the kernels that stream
constexpr int kMaxTileGroups = 64;  // groups per tile of the kernels that hold a tile in registers
constexpr int kMaxStreamGroups = 2048;  // groups per tile of the kernels that stream (kBlock vectors of 8 channels)

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

struct GroupNormArgs {
    const void* x;            // or null: codes and scales of an 8-bit checkpoint
    const signed char* codes;
    const float* scales;
    const void* gamma;        // null: ones
    const void* beta;         // null: zeros
    const void* out_grad;     // backward
    void* out;                // out, or x_grad
    float* stats;             // [samples][groups]: mean, rstd
    float* partial;           // work area
    float* sums;              // backward, work area: [samples][groups] pairs
    u64 positions, rows;      // rows: positions a workgroup of a streaming kernel takes
    u64 x_pitch, grad_pitch, out_pitch;
    unsigned int samples, channels, groups, per_group, tile_groups, tiles, splits;
    unsigned int per_group_magic;  // ceil(2^32 / per_group), for divisions of numbers below 2^16
    int param_f32, activation, accumulate;
    float eps;
};

// e / per_group for e * per_group < 2^32 (0: per_group is 1).
__device__ __forceinline__ unsigned int group_of(unsigned int e, unsigned int magic) {
    return magic ? __umulhi(e, magic) : e;
}

template <class T>
__device__ __forceinline__ float param(const void* p, int f32, unsigned int i, float none) {
    if (!p) return none;
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
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
        return s * (1.0f + z * (1.0f - s));
    }
    if (ACT == kGelu)
        return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * (0.39894228f * __builtin_amdgcn_exp2f(z * z * -0.72134752f));
    return 1.0f;
}
template <class F>
__device__ __forceinline__ void with_activation(int activation, F f) {
    switch (activation) {
        case kRelu: f(std::integral_constant<int, kRelu>()); break;
        case kSilu: f(std::integral_constant<int, kSilu>()); break;
        case kGelu: f(std::integral_constant<int, kGelu>()); break;
        default: f(std::integral_constant<int, kNone>()); break;
    }
}

// Which part of the data a thread of a tile works on: a vector of V channels, the same for all its rows.
// The last vector of a row of W channels starts at W - V; its first `dup` channels are also the vector
// before it's: loaded, but neither summed nor stored here.
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
    Pack<T, V> p;
    __device__ __forceinline__ void load(const GroupNormArgs& a, u64 row, unsigned int channel) {
        p = load_pack<false, T, V>(static_cast<const T*>(a.x) + row * a.x_pitch + channel);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < V; j++) p.v[j] = from_f32<T>(0.0f);
    }
    __device__ __forceinline__ float value(int j) const { return to_f32(p.v[j]); }
};
template <class T, int V>
struct Source<T, V, true> {
    Pack<signed char, V> c;
    float low, high;  // the vector may end in the next block of 128
    int in_low;
    __device__ __forceinline__ void load(const GroupNormArgs& a, u64 row, unsigned int channel) {
        const u64 i = row * a.channels + channel;
        c = load_pack<false, signed char, V>(a.codes + i);
        in_low = 128 - static_cast<int>(i & 127);
        low = a.scales[i >> 7];
        high = in_low < V ? a.scales[(i >> 7) + 1] : low;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < V; j++) c.v[j] = 0;
        low = high = 0.0f;
        in_low = V;
    }
    __device__ __forceinline__ float value(int j) const {
        const float v = static_cast<float>(c.v[j]) * (j < in_low ? low : high);
        return c.v[j] == -128 ? __builtin_nanf("") : v;
    }
};

template <class T, int V>
__device__ __forceinline__ void store_valid(T* p, const Pack<T, V>& pack, int dup) {
    if (dup == 0) {
        store_pack<false, T, V>(p, pack);
    } else {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j >= dup) p[j] = pack.v[j];
    }
}

// Sums of a table of `rows` x `width` floats over the rows and channels of each group; result for group g in
// out[g].  All threads of the workgroup call it; `table` is complete when it is called and free when it
// returns, `out` may be read then.
template <int THREADS>
__device__ __forceinline__ void group_sums(const float* table, unsigned int rows, unsigned int width, unsigned int n_groups,
                                           unsigned int per_group, unsigned int magic, float* wave_sums, float* out) {
    constexpr unsigned int kWaves = THREADS / 64;
    const unsigned int t = threadIdx.x, entries = rows * per_group;
    __syncthreads();
    if (n_groups < kWaves) {
        // several wavefronts per group
        const unsigned int per = kWaves / n_groups, wave = t / 64, g = wave / per;
        float s = 0.0f;
        if (g < n_groups)
            for (unsigned int e = (wave % per) * 64 + t % 64; e < entries; e += per * 64) {
                const unsigned int r = group_of(e, magic);
                s += table[r * width + g * per_group + (e - r * per_group)];
            }
        s = lanes_sum<64>(s);
        if (t % 64 == 0) wave_sums[wave] = s;
        __syncthreads();
        if (t < n_groups) {
            float total = 0.0f;
            for (unsigned int i = 0; i < per; i++) total += wave_sums[t * per + i];
            out[t] = total;
        }
    } else {
        // several groups per wavefront: a power of two of lanes for each
        int lanes = 64;
        while (static_cast<unsigned int>(lanes) * n_groups > THREADS && lanes > 1) lanes /= 2;
        for (unsigned int base = 0; base < n_groups; base += THREADS / lanes) {
            const unsigned int g = base + t / lanes;
            float s = 0.0f;
            if (g < n_groups)
                for (unsigned int e = t % lanes; e < entries; e += lanes) {
                    const unsigned int r = group_of(e, magic);
                    s += table[r * width + g * per_group + (e - r * per_group)];
                }
            s = lanes_sum_of(s, lanes);
            if (g < n_groups && t % lanes == 0) out[g] = s;
        }
    }
    __syncthreads();
}

// Sum over the workgroup, in every thread.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* wave_sums) {
    v = lanes_sum<64>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) wave_sums[threadIdx.x / 64] = v;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) total += wave_sums[w];
    return total;
}

// ---- forward, a tile in registers: one launch, x read once ----

template <class T, int V, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS) custos_group_norm_tile(const GroupNormArgs a) {
    __shared__ float table[THREADS * V];
    __shared__ float wave_sums[THREADS / 64];
    __shared__ float mean_of[kMaxTileGroups], rstd_of[kMaxTileGroups];
    const unsigned int t = threadIdx.x;
    const unsigned int n = blockIdx.x / a.tiles, tile = blockIdx.x - n * a.tiles;
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const unsigned int step = THREADS / vecs;  // rows at a time (the host made sure that it is at least one)
    const unsigned int r0 = t / vecs;
    const Column c = column_of<V>(a, t - r0 * vecs);
    const bool active = r0 < step;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    const u64 row0 = static_cast<u64>(n) * a.positions;
    Source<T, V, false> held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const u64 p = r0 + static_cast<u64>(i) * step;
        if (active && p < a.positions) held[i].load(a, row0 + p, c0 + c.first);
        else held[i].zero();
    }
    const float count = static_cast<float>(a.positions) * static_cast<float>(a.per_group);
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < HELD; i++) sum[j] += held[i].value(j);
        if (active && j >= c.dup) table[r0 * c.width + c.first + j] = sum[j];
    }
    group_sums<THREADS>(table, step, c.width, a.tile_groups, a.per_group, a.per_group_magic, wave_sums, mean_of);
    float mean[V], rstd[V];
#pragma unroll
    for (int j = 0; j < V; j++) mean[j] = mean_of[group_of(c.first + j, a.per_group_magic)] / count;
#pragma unroll
    for (int j = 0; j < V; j++) {
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const float d = held[i].value(j) - mean[j];
            if (r0 + static_cast<u64>(i) * step < a.positions) sum[j] += d * d;
        }
        if (active && j >= c.dup) table[r0 * c.width + c.first + j] = sum[j];
    }
    group_sums<THREADS>(table, step, c.width, a.tile_groups, a.per_group, a.per_group_magic, wave_sums, rstd_of);
#pragma unroll
    for (int j = 0; j < V; j++) rstd[j] = 1.0f / sqrtf(rstd_of[group_of(c.first + j, a.per_group_magic)] / count + a.eps);
    if (t < a.tile_groups) {
        float* s = a.stats + (static_cast<u64>(n) * a.groups + tile * a.tile_groups + t) * 2;
        s[0] = mean_of[t] / count;
        s[1] = 1.0f / sqrtf(rstd_of[t] / count + a.eps);
    }
    if (!active) return;
    float gamma[V], beta[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        gamma[j] = param<T>(a.gamma, a.param_f32, c0 + c.first + j, 1.0f);
        beta[j] = param<T>(a.beta, a.param_f32, c0 + c.first + j, 0.0f);
    }
    T* out = static_cast<T*>(a.out) + row0 * a.out_pitch + c0 + c.first;
    with_activation(a.activation, [&](auto which) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const u64 p = r0 + static_cast<u64>(i) * step;
            if (p >= a.positions) break;
            Pack<T, V> y;
#pragma unroll
            for (int j = 0; j < V; j++)
                y.v[j] = from_f32<T>(act<decltype(which)::value>((held[i].value(j) - mean[j]) * rstd[j] * gamma[j] + beta[j]));
            store_valid<T, V>(out + p * a.out_pitch, y, c.dup);
        }
    });
}

// ---- forward, streaming: parts of every group, the parts joined, the values ----

// Mean and sum of squared distances of every group over the rows of one part.
template <class T, int V>
__global__ void __launch_bounds__(kBlock) custos_group_norm_parts(const GroupNormArgs a) {
    __shared__ float table[kBlock * V];
    __shared__ float wave_sums[kBlock / 64];
    __shared__ float group[kMaxStreamGroups];
    const unsigned int t = threadIdx.x;
    const unsigned int part = blockIdx.x / a.tiles, tile = blockIdx.x - part * a.tiles;
    const unsigned int n = part / a.splits, split = part - n * a.splits;
    const u64 p0 = split * a.rows, p1 = min(p0 + a.rows, a.positions);
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const bool one_column = vecs <= kBlock;
    const unsigned int step = one_column ? kBlock / vecs : 1;
    const unsigned int r0 = one_column ? t / vecs : 0;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    const u64 row0 = static_cast<u64>(n) * a.positions;
    const u64 rows = r0 < step && p0 + r0 < p1 ? (p1 - p0 - r0 + step - 1) / step : 0;
    float* out = a.partial + (static_cast<u64>(part) * a.groups + tile * a.tile_groups) * 2;
    // of the thread, over all its columns (one group per tile), or of its column
    float all = 0.0f, all_mean = 0.0f, all_m2 = 0.0f;
    float mean[V], m2[V];
    Column c = column_of<V>(a, one_column ? t - r0 * vecs : t);
    for (unsigned int col = one_column ? t - r0 * vecs : t; col < vecs && r0 < step; col += kBlock) {
        c = column_of<V>(a, col);
        const u64 first = row0 + p0 + r0;
        float shift[V], s[V], q[V];
#pragma unroll
        for (int j = 0; j < V; j++) shift[j] = s[j] = q[j] = mean[j] = m2[j] = 0.0f;
        if (rows > 0) {
            Source<T, V, false> x;
            x.load(a, first, c0 + c.first);
#pragma unroll
            for (int j = 0; j < V; j++) shift[j] = x.value(j);
        }
        constexpr int kAhead = 4;
        u64 i = 0;
        for (; i + kAhead <= rows; i += kAhead) {
            Source<T, V, false> x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) x[u].load(a, first + (i + u) * step, c0 + c.first);
#pragma unroll
            for (int u = 0; u < kAhead; u++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = x[u].value(j) - shift[j];
                    s[j] += d;
                    q[j] = __builtin_fmaf(d, d, q[j]);
                }
        }
        for (; i < rows; i++) {
            Source<T, V, false> x;
            x.load(a, first + i * step, c0 + c.first);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = x.value(j) - shift[j];
                s[j] += d;
                q[j] = __builtin_fmaf(d, d, q[j]);
            }
        }
        if (rows > 0) {
            const float count = static_cast<float>(rows);
#pragma unroll
            for (int j = 0; j < V; j++) {
                mean[j] = shift[j] + s[j] / count;
                m2[j] = fmaxf(q[j] - s[j] * (s[j] / count), 0.0f);
            }
        }
        if (a.tile_groups == 1 && rows > 0) {
            // the column's channels are one group's: count, mean and squared distances of the thread
            const float count = static_cast<float>(rows) * static_cast<float>(V - c.dup);
            float m = 0.0f, d2 = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) m += j >= c.dup ? mean[j] : 0.0f;
            m /= static_cast<float>(V - c.dup);
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j >= c.dup) d2 += m2[j] + static_cast<float>(rows) * (mean[j] - m) * (mean[j] - m);
            const float both = all + count, delta = m - all_mean;
            all_m2 += d2 + delta * delta * (all * (count / both));
            all_mean += delta * (count / both);
            all = both;
        }
    }
    const float total = static_cast<float>(p1 - p0) * static_cast<float>(a.per_group);
    if (a.tile_groups == 1) {
        const float m = block_sum<kBlock>(all * all_mean, wave_sums) / total;
        const float d2 = block_sum<kBlock>(all_m2 + all * (all_mean - m) * (all_mean - m), wave_sums);
        if (t == 0) out[0] = m, out[1] = d2;
        return;
    }
    const bool active = r0 < step;
#pragma unroll
    for (int j = 0; j < V; j++)
        if (active && j >= c.dup) table[r0 * c.width + c.first + j] = static_cast<float>(rows) * mean[j];
    group_sums<kBlock>(table, step, c.width, a.tile_groups, a.per_group, a.per_group_magic, wave_sums, group);
    for (unsigned int g = t; g < a.tile_groups; g += kBlock) out[g * 2] = group[g] / total;
#pragma unroll
    for (int j = 0; j < V; j++)
        if (active && j >= c.dup) {
            const float d = mean[j] - group[group_of(c.first + j, a.per_group_magic)] / total;
            table[r0 * c.width + c.first + j] = m2[j] + static_cast<float>(rows) * d * d;
        }
    __syncthreads();  // (every thread has read `group`)
    group_sums<kBlock>(table, step, c.width, a.tile_groups, a.per_group, a.per_group_magic, wave_sums, group);
    for (unsigned int g = t; g < a.tile_groups; g += kBlock) out[g * 2 + 1] = group[g];
}

// The parts of a group joined, one wavefront for each: lanes over the parts, sums in f64.
__global__ void __launch_bounds__(kBlock) custos_group_norm_stats(const GroupNormArgs a) {
    const u64 which = static_cast<u64>(blockIdx.x) * (kBlock / 64) + threadIdx.x / 64;
    if (which >= static_cast<u64>(a.samples) * a.groups) return;
    const unsigned int lane = threadIdx.x % 64;
    const u64 n = which / a.groups, g = which - n * a.groups;
    const float* part = a.partial + (n * a.splits * a.groups + g) * 2;
    auto count = [&](unsigned int s) { return static_cast<double>(min(a.rows, a.positions - s * a.rows)) * a.per_group; };
    double sum = 0.0;
    for (unsigned int s = lane; s < a.splits; s += 64) sum += count(s) * part[static_cast<u64>(s) * a.groups * 2];
    const double total = static_cast<double>(a.positions) * a.per_group;
    const double mean = lanes_sum_f64(sum) / total;
    double m2 = 0.0;
    for (unsigned int s = lane; s < a.splits; s += 64) {
        const double d = part[static_cast<u64>(s) * a.groups * 2] - mean;
        m2 += part[static_cast<u64>(s) * a.groups * 2 + 1] + count(s) * d * d;
    }
    m2 = lanes_sum_f64(m2);
    if (lane == 0) {
        a.stats[which * 2] = static_cast<float>(mean);
        a.stats[which * 2 + 1] = static_cast<float>(1.0 / sqrt(m2 / total + static_cast<double>(a.eps)));
    }
}

// What a thread needs of its column's channels.
template <class T, int V>
struct ChannelParams {
    float mean[V], rstd[V], gamma[V], beta[V];
    __device__ __forceinline__ void load(const GroupNormArgs& a, unsigned int n, unsigned int tile, const Column& c) {
        const unsigned int c0 = tile * a.tile_groups * a.per_group;
        const float* stats = a.stats + (static_cast<u64>(n) * a.groups + tile * a.tile_groups) * 2;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const unsigned int g = a.tile_groups == 1 ? 0 : group_of(c.first + j, a.per_group_magic);
            mean[j] = stats[g * 2];
            rstd[j] = stats[g * 2 + 1];
            gamma[j] = param<T>(a.gamma, a.param_f32, c0 + c.first + j, 1.0f);
            beta[j] = param<T>(a.beta, a.param_f32, c0 + c.first + j, 0.0f);
        }
    }
};

template <class T, int V>
__global__ void __launch_bounds__(kBlock) custos_group_norm_values(const GroupNormArgs a) {
    const unsigned int t = threadIdx.x;
    const unsigned int part = blockIdx.x / a.tiles, tile = blockIdx.x - part * a.tiles;
    const unsigned int n = part / a.splits, split = part - n * a.splits;
    const u64 p0 = split * a.rows, p1 = min(p0 + a.rows, a.positions);
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const bool one_column = vecs <= kBlock;
    const unsigned int step = one_column ? kBlock / vecs : 1;
    const unsigned int r0 = one_column ? t / vecs : 0;
    if (r0 >= step || p0 + r0 >= p1) return;
    const u64 rows = (p1 - p0 - r0 + step - 1) / step;
    const u64 first = static_cast<u64>(n) * a.positions + p0 + r0;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    for (unsigned int col = one_column ? t - r0 * vecs : t; col < vecs; col += kBlock) {
        const Column c = column_of<V>(a, col);
        ChannelParams<T, V> k;
        k.load(a, n, tile, c);
        T* out = static_cast<T*>(a.out) + c0 + c.first;
        with_activation(a.activation, [&](auto which) {
            constexpr int kAct = decltype(which)::value;
            auto value = [&](const Source<T, V, false>& x) {
                Pack<T, V> y;
#pragma unroll
                for (int j = 0; j < V; j++)
                    y.v[j] = from_f32<T>(act<kAct>((x.value(j) - k.mean[j]) * k.rstd[j] * k.gamma[j] + k.beta[j]));
                return y;
            };
            constexpr int kAhead = 4;
            u64 i = 0;
            for (; i + kAhead <= rows; i += kAhead) {
                Source<T, V, false> x[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) x[u].load(a, first + (i + u) * step, c0 + c.first);
#pragma unroll
                for (int u = 0; u < kAhead; u++) store_valid<T, V>(out + (first + (i + u) * step) * a.out_pitch, value(x[u]), c.dup);
            }
            for (; i < rows; i++) {
                Source<T, V, false> x;
                x.load(a, first + i * step, c0 + c.first);
                store_valid<T, V>(out + (first + i * step) * a.out_pitch, value(x), c.dup);
            }
        });
    }
}

// ---- backward ----
//
// Work area: for every sample and part [2][channels] sums of dz and of dz * h (`partial`); joined over the
// parts, [samples][2][channels] (in the place of part 0); and [samples][groups] pairs of the two means over a group (`sums`).

// dz and h of one element.
template <int ACT>
__device__ __forceinline__ float dz_of(float x, float out_grad, float mean, float rstd, float gamma, float beta, float* h) {
    *h = (x - mean) * rstd;
    const float z = *h * gamma + beta;
    return out_grad * act_grad<ACT>(z);
}

template <class T, int V>
__device__ __forceinline__ void store_grad(const GroupNormArgs& a, T* p, float (&g)[V], int dup) {
    Pack<T, V> y;
    if (a.accumulate) {
        const Pack<T, V> was = load_pack<false, T, V>(p);
#pragma unroll
        for (int j = 0; j < V; j++) g[j] += to_f32(was.v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; j++) y.v[j] = from_f32<T>(g[j]);
    store_valid<T, V>(p, y, dup);
}

// A tile in registers: x and out_grad read once.
template <class T, int V, int HELD, int THREADS, bool SAVED>
__global__ void __launch_bounds__(THREADS) custos_group_norm_grad_tile(const GroupNormArgs a) {
    __shared__ float table[THREADS * V];
    __shared__ float wave_sums[THREADS / 64];
    __shared__ float sum_dh[kMaxTileGroups], sum_dhh[kMaxTileGroups];
    const unsigned int t = threadIdx.x;
    const unsigned int n = blockIdx.x / a.tiles, tile = blockIdx.x - n * a.tiles;
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const unsigned int step = THREADS / vecs;
    const unsigned int r0 = t / vecs;
    const Column c = column_of<V>(a, t - r0 * vecs);
    const bool active = r0 < step;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    const u64 row0 = static_cast<u64>(n) * a.positions;
    const T* out_grad = static_cast<const T*>(a.out_grad) + row0 * a.grad_pitch + c0 + c.first;
    Source<T, V, SAVED> held[HELD];
    Pack<T, V> grad[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const u64 p = r0 + static_cast<u64>(i) * step;
        if (active && p < a.positions) {
            held[i].load(a, row0 + p, c0 + c.first);
            grad[i] = load_pack<false, T, V>(out_grad + p * a.grad_pitch);
        } else {
            held[i].zero();
#pragma unroll
            for (int j = 0; j < V; j++) grad[i].v[j] = from_f32<T>(0.0f);
        }
    }
    ChannelParams<T, V> k;
    k.load(a, n, tile, c);
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.0f;
    with_activation(a.activation, [&](auto which) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            if (r0 + static_cast<u64>(i) * step >= a.positions) break;
#pragma unroll
            for (int j = 0; j < V; j++) {
                float h;
                const float dz = dz_of<decltype(which)::value>(held[i].value(j), to_f32(grad[i].v[j]), k.mean[j], k.rstd[j],
                                                               k.gamma[j], k.beta[j], &h);
                s1[j] += dz;
                s2[j] = __builtin_fmaf(dz, h, s2[j]);
            }
        }
    });
    // over the rows of the workgroup: per channel, which is what the gradients of gamma and beta need, and
    // from there per group
    float* channel = a.partial + static_cast<u64>(n) * 2 * a.channels + c0;
    for (int which = 0; which < 2; which++) {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (active && j >= c.dup) table[r0 * c.width + c.first + j] = which ? s2[j] : s1[j];
        __syncthreads();
        for (unsigned int ch = t; ch < c.width; ch += THREADS) {
            float s = 0.0f;
            for (unsigned int r = 0; r < step; r++) s += table[r * c.width + ch];
            channel[static_cast<u64>(which) * a.channels + ch] = s;
            table[ch] = s * param<T>(a.gamma, a.param_f32, c0 + ch, 1.0f);
        }
        group_sums<THREADS>(table, 1, c.width, a.tile_groups, a.per_group, a.per_group_magic, wave_sums, which ? sum_dhh : sum_dh);
    }
    if (!a.out || !active) return;
    const float count = static_cast<float>(a.positions) * static_cast<float>(a.per_group);
    float mean_dh[V], mean_dhh[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const unsigned int g = group_of(c.first + j, a.per_group_magic);
        mean_dh[j] = sum_dh[g] / count;
        mean_dhh[j] = sum_dhh[g] / count;
    }
    T* out = static_cast<T*>(a.out) + row0 * a.out_pitch + c0 + c.first;
    with_activation(a.activation, [&](auto which) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const u64 p = r0 + static_cast<u64>(i) * step;
            if (p >= a.positions) break;
            float g[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                float h;
                const float dz = dz_of<decltype(which)::value>(held[i].value(j), to_f32(grad[i].v[j]), k.mean[j], k.rstd[j],
                                                               k.gamma[j], k.beta[j], &h);
                g[j] = k.rstd[j] * (dz * k.gamma[j] - mean_dh[j] - h * mean_dhh[j]);
            }
            store_grad<T, V>(a, out + p * a.out_pitch, g, c.dup);
        }
    });
}

// Sums of dz and dz * h per channel over the rows of one part.
template <class T, int V, bool SAVED>
__global__ void __launch_bounds__(kBlock) custos_group_norm_grad_parts(const GroupNormArgs a) {
    __shared__ float table[kBlock * V];
    const unsigned int t = threadIdx.x;
    const unsigned int part = blockIdx.x / a.tiles, tile = blockIdx.x - part * a.tiles;
    const unsigned int n = part / a.splits, split = part - n * a.splits;
    const u64 p0 = split * a.rows, p1 = min(p0 + a.rows, a.positions);
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const bool one_column = vecs <= kBlock;
    const unsigned int step = one_column ? kBlock / vecs : 1;
    const unsigned int r0 = one_column ? t / vecs : 0;
    const u64 rows = r0 < step && p0 + r0 < p1 ? (p1 - p0 - r0 + step - 1) / step : 0;
    const u64 first = static_cast<u64>(n) * a.positions + p0 + r0;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    float* channel = a.partial + static_cast<u64>(part) * 2 * a.channels + c0;
    float s1[V], s2[V];
    Column c = column_of<V>(a, one_column ? t - r0 * vecs : t);
    for (unsigned int col = one_column ? t - r0 * vecs : t; col < vecs && r0 < step; col += kBlock) {
        c = column_of<V>(a, col);
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.0f;
        ChannelParams<T, V> k;
        k.load(a, n, tile, c);
        const T* out_grad = static_cast<const T*>(a.out_grad) + c0 + c.first;
        with_activation(a.activation, [&](auto which) {
            auto add = [&](const Source<T, V, SAVED>& x, const Pack<T, V>& g) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<decltype(which)::value>(x.value(j), to_f32(g.v[j]), k.mean[j], k.rstd[j], k.gamma[j],
                                                                   k.beta[j], &h);
                    s1[j] += dz;
                    s2[j] = __builtin_fmaf(dz, h, s2[j]);
                }
            };
            constexpr int kAhead = 2;
            u64 i = 0;
            for (; i + kAhead <= rows; i += kAhead) {
                Source<T, V, SAVED> x[kAhead];
                Pack<T, V> g[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const u64 row = first + (i + u) * step;
                    x[u].load(a, row, c0 + c.first);
                    g[u] = load_pack<false, T, V>(out_grad + row * a.grad_pitch);
                }
#pragma unroll
                for (int u = 0; u < kAhead; u++) add(x[u], g[u]);
            }
            for (; i < rows; i++) {
                Source<T, V, SAVED> x;
                x.load(a, first + i * step, c0 + c.first);
                add(x, load_pack<false, T, V>(out_grad + (first + i * step) * a.grad_pitch));
            }
        });
        if (!one_column) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j >= c.dup) channel[c.first + j] = s1[j], channel[a.channels + c.first + j] = s2[j];
        }
    }
    if (!one_column) return;
    const bool active = r0 < step;
    for (int which = 0; which < 2; which++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; j++)
            if (active && j >= c.dup) table[r0 * c.width + c.first + j] = which ? s2[j] : s1[j];
        __syncthreads();
        for (unsigned int ch = t; ch < c.width; ch += kBlock) {
            float s = 0.0f;
            for (unsigned int r = 0; r < step; r++) s += table[r * c.width + ch];
            channel[static_cast<u64>(which) * a.channels + ch] = s;
        }
    }
}

// The parts of a sample joined, one workgroup for every sample and group: per channel (over the part 0 sums),
// and the two means over the group.
template <class T>
__global__ void __launch_bounds__(kBlock) custos_group_norm_grad_sums(const GroupNormArgs a) {
    __shared__ float table[2 * kBlock];
    __shared__ float wave_sums[kBlock / 64];
    const unsigned int t = threadIdx.x;
    const unsigned int n = blockIdx.x / a.groups, g = blockIdx.x - n * a.groups;
    const unsigned int c0 = g * a.per_group;
    float* part = a.partial + static_cast<u64>(n) * a.splits * 2 * a.channels + c0;
    float dh = 0.0f, dhh = 0.0f;
    // (threads over the channels, and over the parts where there are fewer channels than threads)
    const unsigned int cols = min(a.per_group, static_cast<unsigned int>(kBlock)), lanes = kBlock / cols;
    const unsigned int r = t / cols;
    for (unsigned int base = 0; base < a.per_group; base += cols) {
        const unsigned int ch = base + (t - r * cols);
        const bool active = r < lanes && ch < a.per_group;
        float s1 = 0.0f, s2 = 0.0f;
        if (active)
            for (unsigned int s = r; s < a.splits; s += lanes) {
                s1 += part[static_cast<u64>(s) * 2 * a.channels + ch];
                s2 += part[(static_cast<u64>(s) * 2 + 1) * a.channels + ch];
            }
        __syncthreads();
        table[t] = s1;
        table[kBlock + t] = s2;
        __syncthreads();
        if (!active || r != 0) continue;
        for (unsigned int l = 1; l < lanes; l++) {
            s1 += table[l * cols + t];
            s2 += table[kBlock + l * cols + t];
        }
        part[ch] = s1;
        part[a.channels + ch] = s2;
        const float gamma = param<T>(a.gamma, a.param_f32, c0 + ch, 1.0f);
        dh += s1 * gamma;
        dhh += s2 * gamma;
    }
    dh = block_sum<kBlock>(dh, wave_sums);
    dhh = block_sum<kBlock>(dhh, wave_sums);
    if (t == 0) {
        const float count = static_cast<float>(a.positions) * static_cast<float>(a.per_group);
        a.sums[(static_cast<u64>(n) * a.groups + g) * 2] = dh / count;
        a.sums[(static_cast<u64>(n) * a.groups + g) * 2 + 1] = dhh / count;
    }
}

template <class T, int V, bool SAVED>
__global__ void __launch_bounds__(kBlock) custos_group_norm_grad_values(const GroupNormArgs a) {
    const unsigned int t = threadIdx.x;
    const unsigned int part = blockIdx.x / a.tiles, tile = blockIdx.x - part * a.tiles;
    const unsigned int n = part / a.splits, split = part - n * a.splits;
    const u64 p0 = split * a.rows, p1 = min(p0 + a.rows, a.positions);
    const unsigned int vecs = (a.tile_groups * a.per_group + V - 1) / V;
    const bool one_column = vecs <= kBlock;
    const unsigned int step = one_column ? kBlock / vecs : 1;
    const unsigned int r0 = one_column ? t / vecs : 0;
    if (r0 >= step || p0 + r0 >= p1) return;
    const u64 rows = (p1 - p0 - r0 + step - 1) / step;
    const u64 first = static_cast<u64>(n) * a.positions + p0 + r0;
    const unsigned int c0 = tile * a.tile_groups * a.per_group;
    const float* sums = a.sums + (static_cast<u64>(n) * a.groups + tile * a.tile_groups) * 2;
    for (unsigned int col = one_column ? t - r0 * vecs : t; col < vecs; col += kBlock) {
        const Column c = column_of<V>(a, col);
        ChannelParams<T, V> k;
        k.load(a, n, tile, c);
        float mean_dh[V], mean_dhh[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const unsigned int g = a.tile_groups == 1 ? 0 : group_of(c.first + j, a.per_group_magic);
            mean_dh[j] = sums[g * 2];
            mean_dhh[j] = sums[g * 2 + 1];
        }
        const T* out_grad = static_cast<const T*>(a.out_grad) + c0 + c.first;
        T* out = static_cast<T*>(a.out) + c0 + c.first;
        with_activation(a.activation, [&](auto which) {
            auto put = [&](u64 row, const Source<T, V, SAVED>& x, const Pack<T, V>& og) {
                float g[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float h;
                    const float dz = dz_of<decltype(which)::value>(x.value(j), to_f32(og.v[j]), k.mean[j], k.rstd[j], k.gamma[j],
                                                                   k.beta[j], &h);
                    g[j] = k.rstd[j] * (dz * k.gamma[j] - mean_dh[j] - h * mean_dhh[j]);
                }
                store_grad<T, V>(a, out + row * a.out_pitch, g, c.dup);
            };
            constexpr int kAhead = 2;
            u64 i = 0;
            for (; i + kAhead <= rows; i += kAhead) {
                Source<T, V, SAVED> x[kAhead];
                Pack<T, V> g[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const u64 row = first + (i + u) * step;
                    x[u].load(a, row, c0 + c.first);
                    g[u] = load_pack<false, T, V>(out_grad + row * a.grad_pitch);
                }
#pragma unroll
                for (int u = 0; u < kAhead; u++) put(first + (i + u) * step, x[u], g[u]);
            }
            for (; i < rows; i++) {
                const u64 row = first + i * step;
                Source<T, V, SAVED> x;
                x.load(a, row, c0 + c.first);
                put(row, x, load_pack<false, T, V>(out_grad + row * a.grad_pitch));
            }
        });
    }
}

// gamma_grad and beta_grad: the channel sums of the samples, added in their order.
__global__ void __launch_bounds__(kBlock) custos_group_norm_param_grads(const float* sums, u64 sample_stride, unsigned int samples,
                                                                        unsigned int channels, float* gamma_grad, float* beta_grad,
                                                                        int accumulate) {
    const unsigned int ch = blockIdx.x * kBlock + threadIdx.x;
    if (ch >= channels) return;
    float s1 = 0.0f, s2 = 0.0f;
    for (unsigned int n = 0; n < samples; n++) {
        s1 += sums[n * sample_stride + ch];
        s2 += sums[n * sample_stride + channels + ch];
    }
    if (beta_grad) beta_grad[ch] = accumulate ? beta_grad[ch] + s1 : s1;
    if (gamma_grad) gamma_grad[ch] = accumulate ? gamma_grad[ch] + s2 : s2;
}

// ---- host ----

struct Plan {
    int vec = 1;                // channels per thread
    bool in_registers = false;
    int threads = kBlock;
    int held = 0;
    GroupNormArgs a{};
};

unsigned int magic_of(unsigned int d) { return d == 1 ? 0u : static_cast<unsigned int>((0x100000000ull + d - 1) / d); }

// The smallest divisor of `groups` whose tile is at least `channels` wide (or all groups); 0: more groups than
// the kernels that hold a tile take.
unsigned int tile_at_least(unsigned int groups, unsigned int per_group, unsigned int channels) {
    for (unsigned int k = 1; k <= std::min<unsigned int>(groups, kMaxTileGroups); k++)
        if (groups % k == 0 && (static_cast<u64>(k) * per_group >= channels || k == groups)) return k;
    return 0;
}
// The largest divisor of `groups` whose rows take at most kBlock vectors (or one group).
unsigned int tile_at_most(unsigned int groups, unsigned int per_group, unsigned int vec) {
    const u64 most = std::min<u64>(groups, static_cast<u64>(kBlock) * vec / per_group);
    for (unsigned int k = static_cast<unsigned int>(most); k > 1; k--)
        if (groups % k == 0) return k;
    return 1;
}

// (threads, vectors held) of the kernels that hold a tile in registers, smallest first.
struct Held {
    int threads, held;
};
constexpr Held kForwardHeld[] = {{256, 4}, {256, 16}, {1024, 16}};
constexpr Held kBackwardHeld[] = {{256, 4}, {1024, 4}};

template <size_t N>
void make_plan(const custos_hip_group_norm_desc& d, size_t elem, const Held (&choices)[N], Plan* plan) {
    GroupNormArgs& a = plan->a;
    a.positions = d.positions;
    a.samples = static_cast<unsigned int>(d.samples);
    a.channels = static_cast<unsigned int>(d.channels);
    a.groups = static_cast<unsigned int>(d.groups);
    a.per_group = a.channels / a.groups;
    a.per_group_magic = magic_of(a.per_group);
    a.activation = d.activation;
    a.eps = static_cast<float>(d.eps);
    const unsigned int full = static_cast<unsigned int>(16 / elem);
    // in registers, if a tile of whole groups of at least 64 bytes a row fits
    {
        const unsigned int k = tile_at_least(a.groups, a.per_group, static_cast<unsigned int>(64 / elem));
        const u64 width = static_cast<u64>(k) * a.per_group;
        const unsigned int vec = width >= full ? full : 1;
        const u64 vecs = (width + vec - 1) / vec;
        for (const Held& h : choices) {
            if (k == 0 || vecs > static_cast<u64>(h.threads)) continue;
            const u64 step = static_cast<u64>(h.threads) / vecs;
            if ((a.positions + step - 1) / step > static_cast<u64>(h.held)) continue;
            plan->in_registers = true;
            plan->vec = static_cast<int>(vec);
            plan->threads = h.threads;
            plan->held = h.held;
            a.tile_groups = k;
            a.tiles = a.groups / k;
            a.splits = 1;
            a.rows = a.positions;
            return;
        }
    }
    plan->vec = static_cast<int>(a.channels >= full ? full : 1);
    a.tile_groups = tile_at_most(a.groups, a.per_group, static_cast<unsigned int>(plan->vec));
    if (static_cast<u64>(a.tile_groups) * a.per_group < static_cast<u64>(plan->vec)) plan->vec = 1;
    a.tiles = a.groups / a.tile_groups;
    const u64 vecs = (static_cast<u64>(a.tile_groups) * a.per_group + plan->vec - 1) / plan->vec;
    const u64 step = std::max<u64>(1, kBlock / vecs);
    // parts: enough workgroups to fill the chip several times, each with a few rounds of rows
    const u64 wanted = std::max<u64>(1, 2048 / (static_cast<u64>(a.samples) * a.tiles));
    const u64 rounds = (a.positions + step - 1) / step;
    u64 splits = std::min<u64>(wanted, std::max<u64>(1, rounds / 8));
    a.rows = (rounds + splits - 1) / splits * step;
    splits = (a.positions + a.rows - 1) / a.rows;
    a.splits = static_cast<unsigned int>(splits);
}

size_t elem_size(int32_t dtype) { return dtype == CUSTOS_HIP_F32 ? 4 : 2; }

int32_t check_desc(custos_hip_device* dev, const char* what, const custos_hip_group_norm_desc* d) {
    auto bad = [&](const char* why) { return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why); };
    if (!d) return bad("the description is null");
    if (d->dtype != CUSTOS_HIP_F32 && d->dtype != CUSTOS_HIP_F16 && d->dtype != CUSTOS_HIP_BF16) return bad("elements are f32, f16 or bf16");
    if (d->param_dtype != CUSTOS_HIP_F32 && d->param_dtype != d->dtype) return bad("gamma and beta are f32 or of the element type");
    if (d->activation < 0 || d->activation > CUSTOS_HIP_ACT_GELU) return bad("unknown activation");
    if (d->flags & ~CUSTOS_HIP_GRAD_OVERWRITE) return bad("unknown flag");
    if (d->channels == 0 || d->groups == 0 || d->channels % d->groups != 0) return bad("the channels divide into the groups");
    if (!(d->eps > 0) || !std::isfinite(d->eps)) return bad("eps is positive");
    if (d->channels >= (1ull << 30) || d->samples >= (1ull << 31) || d->positions >= (1ull << 40) ||
        static_cast<double>(d->samples) * static_cast<double>(d->positions) * static_cast<double>(d->channels) > 1e15)
        return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": the sizes are beyond any memory");
    return CUSTOS_HIP_OK;
}

int32_t check_grid(custos_hip_device* dev, const char* what, u64 blocks) {
    if (blocks >= (1ull << 31)) return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": more than 2^31 workgroups");
    return CUSTOS_HIP_OK;
}

template <class K>
void* handle(K* kernel) {
    return reinterpret_cast<void*>(kernel);
}

struct Kernel {
    void* fn;
    const char* name;
};

template <class T>
Kernel forward_tile(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_tile";
    const bool wide = p.vec > 1;
    if (p.threads == 1024) return {wide ? handle(custos_group_norm_tile<T, V, 16, 1024>) : handle(custos_group_norm_tile<T, 1, 16, 1024>), name};
    if (p.held == 16) return {wide ? handle(custos_group_norm_tile<T, V, 16, 256>) : handle(custos_group_norm_tile<T, 1, 16, 256>), name};
    return {wide ? handle(custos_group_norm_tile<T, V, 4, 256>) : handle(custos_group_norm_tile<T, 1, 4, 256>), name};
}
template <class T>
Kernel forward_parts(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_parts<T, V>) : handle(custos_group_norm_parts<T, 1>), "custos_group_norm_parts"};
}
template <class T>
Kernel forward_values(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_values<T, V>) : handle(custos_group_norm_values<T, 1>), "custos_group_norm_values"};
}
template <class T, bool SAVED>
Kernel backward_tile(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    const char* name = "custos_group_norm_grad_tile";
    const bool wide = p.vec > 1;
    if (p.threads == 1024)
        return {wide ? handle(custos_group_norm_grad_tile<T, V, 4, 1024, SAVED>) : handle(custos_group_norm_grad_tile<T, 1, 4, 1024, SAVED>), name};
    return {wide ? handle(custos_group_norm_grad_tile<T, V, 4, 256, SAVED>) : handle(custos_group_norm_grad_tile<T, 1, 4, 256, SAVED>), name};
}
template <class T, bool SAVED>
Kernel backward_parts(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_grad_parts<T, V, SAVED>) : handle(custos_group_norm_grad_parts<T, 1, SAVED>),
            "custos_group_norm_grad_parts"};
}
template <class T, bool SAVED>
Kernel backward_values(const Plan& p) {
    constexpr int V = VecOf<T>::elems;
    return {p.vec > 1 ? handle(custos_group_norm_grad_values<T, V, SAVED>) : handle(custos_group_norm_grad_values<T, 1, SAVED>),
            "custos_group_norm_grad_values"};
}
template <class T>
Kernel backward_sums() {
    return {handle(custos_group_norm_grad_sums<T>), "custos_group_norm_grad_sums"};
}

// `pick<T>()` for the element type
template <class F>
Kernel by_type(int32_t dtype, F pick) {
    if (dtype == CUSTOS_HIP_F32) return pick(float());
    if (dtype == CUSTOS_HIP_F16) return pick(static_cast<_Float16>(0));
    return pick(static_cast<__bf16>(0));
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
    Operand ops[5] = {{"out", out, rows, desc->channels * es, out_pitch * es, true, es},
                      {"stats", stats, 1, desc->samples * desc->groups * 8, 0, true, 4},
                      {"x", x, rows, desc->channels * es, x_pitch * es, false, es}};
    size_t n = 3;
    if (gamma) ops[n++] = {"gamma", gamma, 1, desc->channels * ps, 0, false, ps};
    if (beta) ops[n++] = {"beta", beta, 1, desc->channels * ps, 0, false, ps};
    rc = check_operands(dev, "group norm", ops, n, /*may_alias=*/true);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);

    Plan plan;
    make_plan(*desc, es, kForwardHeld, &plan);
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
    const u64 parts = static_cast<u64>(a.samples) * a.splits, blocks = parts * a.tiles;
    rc = check_grid(dev, "group norm", blocks);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (plan.in_registers)
        return launch(dev, by_type(desc->dtype, [&](auto t) { return forward_tile<decltype(t)>(plan); }), blocks, plan.threads, a, acc, n);

    const size_t bytes = parts * a.groups * 2 * sizeof(float);
    uint64_t area = 0;
    rc = operator_workspace(dev, bytes, &area);
    if (rc != CUSTOS_HIP_OK) return rc;
    a.partial = reinterpret_cast<float*>(area);
    const Access area_written{area, area + bytes, true}, area_read{area, area + bytes, false};
    const Access in_parts[2] = {ops[2].access(), area_written};
    rc = launch(dev, by_type(desc->dtype, [&](auto t) { return forward_parts<decltype(t)>(plan); }), blocks, kBlock, a, in_parts, 2);
    if (rc != CUSTOS_HIP_OK) return rc;
    const Access in_stats[2] = {area_read, ops[1].access()};
    const u64 waves = static_cast<u64>(a.samples) * a.groups;
    rc = launch(dev, {handle(custos_group_norm_stats), "custos_group_norm_stats"}, (waves + kBlock / 64 - 1) / (kBlock / 64), kBlock, a, in_stats, 2);
    if (rc != CUSTOS_HIP_OK) return rc;
    acc[1].write = false;  // (the values read the statistics)
    return launch(dev, by_type(desc->dtype, [&](auto t) { return forward_values<decltype(t)>(plan); }), blocks, kBlock, a, acc, n);
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
    if (x_grad) ops[n++] = {"x_grad", x_grad, rows, desc->channels * es, x_grad_pitch * es, true, es};
    const size_t values_written = n;
    if (gamma_grad) ops[n++] = {"gamma_grad", gamma_grad, 1, desc->channels * 4, 0, true, 4};
    if (beta_grad) ops[n++] = {"beta_grad", beta_grad, 1, desc->channels * 4, 0, true, 4};
    const size_t first_read = n;
    ops[n++] = {"out_grad", out_grad, rows, desc->channels * es, out_grad_pitch * es, false, es};
    if (saved) {
        ops[n++] = {"codes", codes, 1, total, 0, false, 1};
        ops[n++] = {"scales", scales, 1, (total + 127) / 128 * 4, 0, false, 4};
    } else {
        ops[n++] = {"x", x, rows, desc->channels * es, x_pitch * es, false, es};
    }
    ops[n++] = {"stats", stats, 1, desc->samples * desc->groups * 8, 0, false, 4};
    if (gamma) ops[n++] = {"gamma", gamma, 1, desc->channels * ps, 0, false, ps};
    if (beta) ops[n++] = {"beta", beta, 1, desc->channels * ps, 0, false, ps};
    static_assert(sizeof ops / sizeof ops[0] >= 9, "three written, six read");
    rc = check_operands(dev, what, ops, n, /*may_alias=*/overwrite);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    if (first_read == 0) return CUSTOS_HIP_OK;  // no gradient is wanted

    Plan plan;
    make_plan(*desc, es, kBackwardHeld, &plan);
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
    const u64 parts = static_cast<u64>(a.samples) * a.splits, blocks = parts * a.tiles;
    rc = check_grid(dev, what, std::max<u64>(blocks, static_cast<u64>(a.samples) * a.groups));
    if (rc != CUSTOS_HIP_OK) return rc;
    const size_t part_bytes = parts * 2 * a.channels * sizeof(float), sum_bytes = static_cast<size_t>(a.samples) * a.groups * 2 * sizeof(float);
    uint64_t area = 0;
    rc = operator_workspace(dev, part_bytes + sum_bytes, &area);
    if (rc != CUSTOS_HIP_OK) return rc;
    a.partial = reinterpret_cast<float*>(area);
    a.sums = reinterpret_cast<float*>(area + part_bytes);
    const Access area_written{area, area + part_bytes + sum_bytes, true}, area_read{area, area + part_bytes + sum_bytes, false};
    Access acc[10];
    size_t n_acc = 0;
    for (size_t i = first_read; i < n; i++) acc[n_acc++] = ops[i].access();
    if (plan.in_registers) {
        for (size_t i = 0; i < values_written; i++) acc[n_acc++] = ops[i].access();
        acc[n_acc++] = area_written;
        rc = launch(dev, by_type(desc->dtype, [&](auto t) { return saved ? backward_tile<decltype(t), true>(plan) : backward_tile<decltype(t), false>(plan); }),
                    blocks, plan.threads, a, acc, n_acc);
        if (rc != CUSTOS_HIP_OK) return rc;
    } else {
        acc[n_acc] = area_written;
        rc = launch(dev, by_type(desc->dtype, [&](auto t) { return saved ? backward_parts<decltype(t), true>(plan) : backward_parts<decltype(t), false>(plan); }),
                    blocks, kBlock, a, acc, n_acc + 1);
        if (rc != CUSTOS_HIP_OK) return rc;
        Access in_sums[2] = {area_written, {}};
        size_t n_sums = 1;
        if (gamma) in_sums[n_sums++] = {gamma, gamma + desc->channels * ps, false};
        rc = launch(dev, by_type(desc->dtype, [&](auto t) { return backward_sums<decltype(t)>(); }), static_cast<u64>(a.samples) * a.groups,
                    kBlock, a, in_sums, n_sums);
        if (rc != CUSTOS_HIP_OK) return rc;
        if (x_grad) {
            acc[n_acc++] = area_read;
            acc[n_acc++] = ops[0].access();
            rc = launch(dev, by_type(desc->dtype, [&](auto t) { return saved ? backward_values<decltype(t), true>(plan) : backward_values<decltype(t), false>(plan); }),
                        blocks, kBlock, a, acc, n_acc);
            if (rc != CUSTOS_HIP_OK) return rc;
        }
    }
    if (!gamma_grad && !beta_grad) return CUSTOS_HIP_OK;
    const u64 stride = static_cast<u64>(a.splits) * 2 * a.channels;
    const float* sums = a.partial;
    float *dgamma = reinterpret_cast<float*>(gamma_grad), *dbeta = reinterpret_cast<float*>(beta_grad);
    const OpArg args[] = {{&sums, 8}, {&stride, 8}, {&a.samples, 4}, {&a.channels, 4}, {&dgamma, 8}, {&dbeta, 8}, {&a.accumulate, 4}};
    Access in_params[3] = {area_read, {}, {}};
    size_t n_params = 1;
    for (size_t i = values_written; i < first_read; i++) in_params[n_params++] = ops[i].access();
    OpLaunch op{};
    op.name = "custos_group_norm_param_grads";
    op.func = handle(custos_group_norm_param_grads);
    op.grid = dim3((a.channels + kBlock - 1) / kBlock);
    op.block = dim3(kBlock);
    op.args = args;
    op.n_args = sizeof args / sizeof args[0];
    op.acc = in_params;
    op.n_acc = n_params;
    return launch_op(dev, op);
}

}  // extern "C"
