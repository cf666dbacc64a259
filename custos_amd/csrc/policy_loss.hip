// Log-probabilities of chosen tokens, and the clipped policy loss with its KL term and its gradient
// (custos_hip_token_logprob, custos_hip_policy_loss in include/custos_hip.h).  No counterpart in the reference.
//
// A row of `vocab` logits z, temperature T, chosen token `label`:
//
//   lse = log sum exp(z / T)          logp = z[label] / T - lse          p = exp(z / T - lse)
//   r = exp(logp - old_logp)          d = ref_logp - logp                kl = exp(d) - 1 - d
//   loss = weight * (kl_coef * kl - min(r A, clamp(r, 1 - low, 1 + high) A))
//   slope = d loss / d logp = weight * (-[r A <= clamp(r) A] r A - kl_coef * (exp(d) - 1))
//   d loss / d z = slope / T * (onehot(label) - p)
//
// The row is read once and held in registers (up to 1024 threads of 16 vectors of 16 bytes), with a running
// maximum and sum on the way in; the gradient is formed from the registers.  Longer rows are read twice, the
// second time mostly from the caches.  Bound by memory, with two exponentials per element close behind
// (the hardware exp2 runs at a quarter of the rate of a multiplication).  4096 rows of 131072 bf16 in 415 us (5.2 TB/s;
// 391 with the arithmetic taken out: a row of 256 KiB fills the registers of a CU, so that nothing loads while a row is
// finished), 1999 of 50021 in 75 (5.3 TB/s), and 4.5 for the totals.
//
// exp((z - max) / T) is taken of the difference, never of z / T: a row of the type's lowest value is a uniform
// distribution, not an overflow.  The handful of values per row is computed in f64, by one wavefront: next to
// the border of the clipping range a ratio decides whether a whole row has a gradient, and exp(d) - 1 - d is a
// small difference.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "op_device.hpp"
#include "runtime.hpp"

namespace custos_hip {

namespace {

struct RowArgs {
    const void* logits;
    const int* labels;
    const float* old_logp;
    const float* ref_logp;  // null: no KL term
    const float* advantages;
    const float* weights;
    void* grad;             // null: not wanted
    float* logp;
    float* lse;             // log-probabilities only; may be null
    float4* terms;          // policy: [rows], the four totals' parts; null: not wanted
    u64 pitch, grad_pitch;
    unsigned int vocab;
    float scale2;           // log2(e) / T
    double inv_t, clip_low, clip_high, kl_coef, grad_factor;  // inv_t: 1 / T
};

enum Mode { kLogprob = 0, kPolicy = 1 };

// Running maximum and sum of exp2((z - max) * scale2); the sum of an empty or all -inf range is 0.
struct Running {
    float max = -__builtin_inff(), sum = 0.0f;
    // what differences are taken from: the maximum, or 0 where there is none
    __device__ __forceinline__ static float base(float m) { return m == -__builtin_inff() ? 0.0f : m; }
    template <int V>
    __device__ __forceinline__ void add(const float (&z)[V], float scale2) {
        float m = max;
#pragma unroll
        for (int j = 0; j < V; j++) m = fmaxf(m, z[j]);
        const float b = base(m);
        float e[V];
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = __builtin_amdgcn_exp2f((z[j] - b) * scale2);
#pragma unroll
        for (int half = V / 2; half > 0; half /= 2)
#pragma unroll
            for (int j = 0; j < half; j++) e[j] += e[j + half];
        sum = sum * __builtin_amdgcn_exp2f((max - b) * scale2) + e[0];
        max = m;
    }
    // over the wavefront, in every lane
    __device__ __forceinline__ void join_lanes(float scale2) {
        float m = max;
#pragma unroll
        for (int step = 32; step > 0; step /= 2) m = fmaxf(m, __shfl_xor(m, step, 64));
        sum = lanes_sum(sum * __builtin_amdgcn_exp2f((max - base(m)) * scale2));
        max = m;
    }
};

// The fewer than V elements of a row before the first 16-byte boundary, or behind the last whole vector: thread 0 has
// the former, the last thread the latter, every other thread none.  What is not there counts as -inf.
template <class T, int V>
struct Edge {
    unsigned int first = 0, count = 0;
    T v[V];
    __device__ __forceinline__ void load(const T* row) {
        if (count == 0) return;
#pragma unroll
        for (int j = 0; j < V - 1; j++) v[j] = static_cast<unsigned int>(j) < count ? row[first + j] : from_f32<T>(-__builtin_inff());
        v[V - 1] = from_f32<T>(-__builtin_inff());
    }
};

template <class T, int V>
__device__ __forceinline__ void add_vector(Running* run, const Pack<T, V>& p, float scale2) {
    float z[V];
#pragma unroll
    for (int j = 0; j < V; j++) z[j] = to_f32(p.v[j]);
    run->add(z, scale2);
}

// What the gradient's elements need: dz = exp * factor, + slope at the label.
struct RowGradient {
    float base, factor, slope;
    int label;
    template <class T, int V>
    __device__ __forceinline__ Pack<T, V> of(const Pack<T, V>& z, unsigned int first, float scale2) const {
        float g[V];
#pragma unroll
        for (int j = 0; j < V; j++) g[j] = __builtin_amdgcn_exp2f((to_f32(z.v[j]) - base) * scale2) * factor;
        const unsigned int at = static_cast<unsigned int>(label) - first;
        if (at < static_cast<unsigned int>(V)) {
#pragma unroll
            for (int j = 0; j < V; j++) g[j] += at == static_cast<unsigned int>(j) ? slope : 0.0f;
        }
        Pack<T, V> y;
#pragma unroll
        for (int j = 0; j < V; j++) y.v[j] = from_f32<T>(g[j]);
        return y;
    }
};

// What a row brings besides its logits.
struct RowInputs {
    int label;
    float z_label, weight, advantage, old_logp, ref_logp;
};

// The few values of a row, by one whole wavefront; lane 0 writes them down.
template <int MODE>
__device__ __forceinline__ void finish_row(const RowArgs& a, u64 row, const RowInputs& in, const Running& run, RowGradient* out) {
    const unsigned int lane = threadIdx.x % 64;
    const double log_sum = log(static_cast<double>(run.sum));
    const bool chosen = in.label >= 0;
    const double logp = (static_cast<double>(in.z_label) - static_cast<double>(run.max)) * a.inv_t - log_sum;
    if (lane == 0 && a.logp) a.logp[row] = chosen ? static_cast<float>(logp) : 0.0f;
    if (MODE == kLogprob) {
        if (lane == 0 && a.lse) a.lse[row] = static_cast<float>(static_cast<double>(run.max) * a.inv_t + log_sum);
        return;
    }
    const double weight = in.weight, advantage = in.advantage;
    const double moved = logp - static_cast<double>(in.old_logp);
    const double behind = a.ref_logp ? static_cast<double>(in.ref_logp) - logp : 0.0;
    // exp - 1 of both differences at once, in two lanes
    const double em1 = expm1(lane == 0 ? moved : behind);
    const double behind_em1 = __shfl(em1, 1, 64);
    double ratio = __shfl(em1, 0, 64) + 1.0;
    if (ratio < 0.5) ratio = exp(moved);  // (the sum cancels: a ratio of e^-30 would have four digits, one of e^-37 none)
    const double kl = behind_em1 - behind;
    const double plain = ratio * advantage;
    const double clipped = fmin(fmax(ratio, 1.0 - a.clip_low), 1.0 + a.clip_high) * advantage;
    const bool inside = !(plain > clipped);  // (a NaN stays one)
    const double value = inside ? plain : clipped;
    const bool counts = a.kl_coef != 0.0;  // (a KL term that is only watched may be infinite: 0 times it is no number)
    if (lane == 0 && a.terms)
        a.terms[row] = make_float4(static_cast<float>(weight * (counts ? a.kl_coef * kl - value : -value)), static_cast<float>(weight * kl),
                                   inside ? 0.0f : in.weight, static_cast<float>(weight * ratio));
    const double slope = weight * ((inside ? -plain : 0.0) - (counts ? a.kl_coef * behind_em1 : 0.0)) * a.grad_factor;
    out->base = Running::base(run.max);
    out->slope = static_cast<float>(slope);
    out->factor = static_cast<float>(-slope / static_cast<double>(run.sum));
    out->label = in.label;
}

// One workgroup per row.  HELD > 0: the row is held in registers, HELD vectors a thread; 0: it is read twice.
// STREAM: the gradient is stored past the caches.
template <class T, int V, int HELD, int THREADS, int MODE, bool STREAM>
__global__ void __launch_bounds__(THREADS) custos_policy_rows(const RowArgs a) {
    constexpr int kWaves = THREADS / 64;
    __shared__ float part_max[kWaves], part_sum[kWaves];
    __shared__ RowGradient shared;
    const unsigned int t = threadIdx.x;
    const u64 row = blockIdx.x;
    const T* z = static_cast<const T*>(a.logits) + row * a.pitch;
    T* grad = MODE == kPolicy && a.grad ? static_cast<T*>(a.grad) + row * a.grad_pitch : nullptr;
    // whole vectors at 16-byte boundaries, from element `head` on, and the edges
    const unsigned int head = min(a.vocab, static_cast<unsigned int>((16 - (reinterpret_cast<u64>(z) & 15)) & 15) / static_cast<unsigned int>(sizeof(T)));
    const unsigned int vecs = (a.vocab - head) / V;
    Edge<T, V> edge;
    if (t == 0) edge.count = head;
    if (t == THREADS - 1) edge.first = head + vecs * V, edge.count = a.vocab - edge.first;
    RowInputs in;
    in.label = a.labels[row];
    if (MODE == kPolicy) {  // (all of them now: nothing waits for them at the end)
        in.weight = a.weights[row];
        in.advantage = a.advantages[row];
        in.old_logp = a.old_logp[row];
        in.ref_logp = a.ref_logp ? a.ref_logp[row] : 0.0f;
    }
    // a row nothing is asked of is not read (but for its first quarter, which is under way when that is known)
    constexpr int kFirst = HELD / 4;
    Bits<T, V> held[HELD > 0 ? HELD : 1];
    auto load_held = [&](int i) {
        const unsigned int v = t + i * THREADS;
        if (v < vecs) held[i].template load<true>(z + head + v * V);
    };
#pragma unroll
    for (int i = 0; i < kFirst; i++) load_held(i);
    if (MODE == kLogprob ? in.label < 0 && !a.lse : in.label < 0 || in.weight == 0.0f) {
        if (t == 0) {
            if (a.logp) a.logp[row] = 0.0f;
            if (MODE == kPolicy && a.terms) a.terms[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        if (grad) {
            Pack<T, V> zero;
#pragma unroll
            for (int j = 0; j < V; j++) zero.v[j] = from_f32<T>(0.0f);
            for (unsigned int v = t; v < vecs; v += THREADS) store_pack<STREAM, T, V>(grad + head + v * V, zero);
            for (unsigned int j = 0; j < edge.count; j++) grad[edge.first + j] = zero.v[0];
        }
        return;
    }
    // (a label behind the vocabulary: NaN, and no read)
    in.z_label = in.label < 0 ? 0.0f : static_cast<unsigned int>(in.label) < a.vocab ? to_f32(z[in.label]) : __builtin_nanf("");
    Running run;
    if (HELD > 0) {
#pragma unroll
        for (int i = kFirst; i < HELD; i++) load_held(i);
        edge.load(z);
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            if (t + i * THREADS >= vecs) break;
            add_vector<T, V>(&run, held[i].pack(), a.scale2);
            held[i].forget_values();
        }
    } else {
        edge.load(z);
        constexpr int kAhead = 4;
        unsigned int v = t;
        for (; v + (kAhead - 1) * THREADS < vecs; v += kAhead * THREADS) {
            Bits<T, V> p[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) p[u].load(z + head + (v + u * THREADS) * V);
#pragma unroll
            for (int u = 0; u < kAhead; u++) add_vector<T, V>(&run, p[u].pack(), a.scale2);
        }
        for (; v < vecs; v += THREADS) add_vector<T, V>(&run, load_pack<false, T, V>(z + head + v * V), a.scale2);
    }
    Pack<T, V> edge_values;
#pragma unroll
    for (int j = 0; j < V; j++) edge_values.v[j] = edge.v[j];
    if (edge.count > 0) add_vector<T, V>(&run, edge_values, a.scale2);
    run.join_lanes(a.scale2);
    if (t % 64 == 0) part_max[t / 64] = run.max, part_sum[t / 64] = run.sum;
    __syncthreads();
    if (t < 64) {
        run.max = t < kWaves ? part_max[t] : -__builtin_inff();
        run.sum = t < kWaves ? part_sum[t] : 0.0f;
        run.join_lanes(a.scale2);
        RowGradient g;
        finish_row<MODE>(a, row, in, run, &g);
        if (MODE == kPolicy && t == 0) shared = g;
    }
    if (MODE == kLogprob || !grad) return;
    __syncthreads();
    const RowGradient g = shared;
    if (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const unsigned int v = t + i * THREADS;
            if (v >= vecs) break;
            store_pack<STREAM, T, V>(grad + head + v * V, g.of<T, V>(held[i].pack(), head + v * V, a.scale2));
        }
    } else {
        for (unsigned int v = t; v < vecs; v += THREADS)
            store_pack<STREAM, T, V>(grad + head + v * V, g.of<T, V>(load_pack<false, T, V>(z + head + v * V), head + v * V, a.scale2));
    }
    if (edge.count > 0) {
        const Pack<T, V> y = g.of<T, V>(edge_values, edge.first, a.scale2);
#pragma unroll
        for (int j = 0; j < V - 1; j++)
            if (static_cast<unsigned int>(j) < edge.count) grad[edge.first + j] = y.v[j];
    }
}

// Sums of rows of four, `rows_each` rows a workgroup, in a fixed order and in f64; to `sums`, of which the next launch
// adds up 8192 again.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) custos_policy_totals(const float4* terms, u64 rows, u64 rows_each, float4* sums) {
    __shared__ double parts[kSumThreads / 64][4];
    const unsigned int t = threadIdx.x;
    const u64 begin = blockIdx.x * rows_each, end = min(begin + rows_each, rows);
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (u64 r = begin + t; r < end; r += kSumThreads) {
        const float4 v = terms[r];
        s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        s[k] = lanes_sum_f64(s[k]);
        if (t % 64 == 0) parts[t / 64][k] = s[k];
    }
    __syncthreads();
    if (t >= 4) return;
    double total = 0.0;
    for (int w = 0; w < kSumThreads / 64; w++) total += parts[w][t];
    reinterpret_cast<float*>(sums + blockIdx.x)[t] = static_cast<float>(total);
}

// ---- host ----

// The gradient of more than 64 MiB moved is stored past the caches, like the second pass of the group norm.
constexpr u64 kStreamBeyond = 64ull << 20;

struct Kernel {
    void* fn;
    int threads;
};

template <class T, int V, int MODE, bool STREAM>
Kernel kernel_for(unsigned int vocab) {
    const u64 vecs = vocab / V;
#define CUSTOS_ROWS(HELD, THREADS) \
    if (HELD == 0 || vecs <= static_cast<u64>(HELD) * THREADS) return {reinterpret_cast<void*>(custos_policy_rows<T, V, HELD, THREADS, MODE, STREAM>), THREADS}
    CUSTOS_ROWS(4, 64);
    CUSTOS_ROWS(4, 256);
    CUSTOS_ROWS(16, 256);
    CUSTOS_ROWS(16, 512);
    CUSTOS_ROWS(16, 1024);
    CUSTOS_ROWS(0, 1024);
#undef CUSTOS_ROWS
}

template <class T, int MODE>
Kernel kernel_of_type(unsigned int vocab, bool stream) {
    constexpr int V = VecOf<T>::elems;
    if (MODE == kPolicy && stream) return kernel_for<T, V, kPolicy, true>(vocab);
    return kernel_for<T, V, MODE, false>(vocab);
}
template <int MODE>
Kernel kernel_of(int32_t dtype, unsigned int vocab, bool stream) {
    if (dtype == CUSTOS_HIP_F32) return kernel_of_type<float, MODE>(vocab, stream);
    if (dtype == CUSTOS_HIP_F16) return kernel_of_type<_Float16, MODE>(vocab, stream);
    return kernel_of_type<__bf16, MODE>(vocab, stream);
}

size_t elem_size(int32_t dtype) { return dtype == CUSTOS_HIP_F32 ? 4 : 2; }

int32_t check_rows(custos_hip_device* dev, const char* what, int32_t dtype, uint64_t rows, uint64_t vocab, double temperature) {
    auto bad = [&](const char* why) { return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why); };
    if (dtype != CUSTOS_HIP_F32 && dtype != CUSTOS_HIP_F16 && dtype != CUSTOS_HIP_BF16) return bad("logits are f32, f16 or bf16");
    if (vocab == 0) return bad("the vocabulary is empty");
    if (!(temperature > 0) || !std::isfinite(temperature) || !std::isfinite(static_cast<float>(1.4426950408889634 / temperature)) ||
        static_cast<float>(1.0 / temperature) == 0.0f)
        return bad("the temperature is positive");
    if (rows >= (1ull << 31) || vocab >= (1ull << 30))
        return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": more than 2^31 rows or 2^30 tokens");
    return CUSTOS_HIP_OK;
}

int32_t launch(custos_hip_device* dev, const char* name, void* fn, u64 blocks, int threads, const OpArg* args, size_t n_args,
               const Access* acc, size_t n_acc) {
    OpLaunch op{};
    op.name = name;
    op.func = fn;
    op.grid = dim3(static_cast<unsigned int>(blocks));
    op.block = dim3(static_cast<unsigned int>(threads));
    op.args = args;
    op.n_args = n_args;
    op.acc = acc;
    op.n_acc = n_acc;
    return launch_op(dev, op);
}

constexpr u64 kRowsEach = 8192;  // rows a workgroup of the totals adds up

int32_t launch_totals(custos_hip_device* dev, uint64_t terms, u64 rows, uint64_t totals) {
    while (true) {
        const u64 blocks = std::max<u64>(1, (rows + kRowsEach - 1) / kRowsEach);
        const uint64_t sums = blocks == 1 ? totals : terms + rows * sizeof(float4);  // (behind the rows they are the sums of)
        const OpArg args[] = {{&terms, 8}, {&rows, 8}, {&kRowsEach, 8}, {&sums, 8}};
        const Access acc[2] = {{terms, terms + rows * sizeof(float4), false}, {sums, sums + blocks * sizeof(float4), true}};
        int32_t rc = launch(dev, "custos_policy_totals", reinterpret_cast<void*>(custos_policy_totals), blocks, kSumThreads, args, 4, acc, 2);
        if (rc != CUSTOS_HIP_OK || blocks == 1) return rc;
        terms = sums;
        rows = blocks;
    }
}

}  // namespace

}  // namespace custos_hip

using namespace custos_hip;

extern "C" {

int32_t custos_hip_token_logprob(custos_hip_device* dev, int32_t dtype, uint64_t logits, uint64_t pitch, uint64_t labels, uint64_t rows,
                                 uint64_t vocab, double temperature, uint64_t logp, uint64_t lse) {
    const char* what = "token log-probabilities";
    int32_t rc = check_rows(dev, what, dtype, rows, vocab, temperature);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (rows == 0) {
        REQUIRE_DEV(dev);
        return CUSTOS_HIP_OK;
    }
    const size_t es = elem_size(dtype);
    Operand ops[4] = {{"logits", logits, rows, vocab * es, pitch * es, false, es},
                      {"labels", labels, 1, rows * 4, 0, false, 4},
                      {"logp", logp, 1, rows * 4, 0, true, 4}};
    size_t n = 3;
    if (lse) ops[n++] = {"lse", lse, 1, rows * 4, 0, true, 4};
    rc = check_operands(dev, what, ops, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    const Kernel k = kernel_of<kLogprob>(dtype, static_cast<unsigned int>(vocab), false);
    rc = check_grid(dev, what, rows, k.threads);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    RowArgs a;
    std::memset(&a, 0, sizeof a);  // (padding included: recordings compare the arguments of their launches byte by byte)
    a.logits = reinterpret_cast<const void*>(logits);
    a.labels = reinterpret_cast<const int*>(labels);
    a.logp = reinterpret_cast<float*>(logp);
    a.lse = reinterpret_cast<float*>(lse);
    a.pitch = pitch;
    a.vocab = static_cast<unsigned int>(vocab);
    a.inv_t = 1.0 / temperature;
    a.scale2 = static_cast<float>(1.4426950408889634 / temperature);
    Access acc[4];
    for (size_t i = 0; i < n; i++) acc[i] = ops[i].access();
    const OpArg arg{&a, sizeof a};
    return launch(dev, "custos_token_logprob", k.fn, rows, k.threads, &arg, 1, acc, n);
}

int32_t custos_hip_policy_loss(custos_hip_device* dev, const custos_hip_policy_desc* desc, uint64_t logits, uint64_t labels, uint64_t old_logp,
                               uint64_t ref_logp, uint64_t advantages, uint64_t weights, uint64_t logits_grad, uint64_t logp, uint64_t totals) {
    const char* what = "policy loss";
    auto bad = [&](const char* why) { return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why); };
    if (!desc) return bad("the description is null");
    int32_t rc = check_rows(dev, what, desc->dtype, desc->rows, desc->vocab, desc->temperature);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (desc->reserved != 0) return bad("the reserved field is zero");
    if (!(desc->clip_low >= 0) || !(desc->clip_low <= 1) || !(desc->clip_high >= 0) || !std::isfinite(desc->clip_high))
        return bad("clip_low is within 0 and 1, clip_high not negative");
    if (!std::isfinite(desc->kl_coef) || !std::isfinite(desc->grad_scale)) return bad("kl_coef and grad_scale are finite");
    if (desc->kl_coef != 0 && !ref_logp) return bad("a KL term needs ref_logp");
    const u64 rows = desc->rows;
    const size_t es = elem_size(desc->dtype);
    Operand ops[9];
    size_t n = 0;
    if (rows > 0) {
        if (logits_grad) ops[n++] = {"logits_grad", logits_grad, rows, desc->vocab * es, desc->grad_pitch * es, true, es, true};
        if (logp) ops[n++] = {"logp", logp, 1, rows * 4, 0, true, 4};
        ops[n++] = {"logits", logits, rows, desc->vocab * es, desc->pitch * es, false, es, true};
        ops[n++] = {"labels", labels, 1, rows * 4, 0, false, 4};
        ops[n++] = {"old_logp", old_logp, 1, rows * 4, 0, false, 4};
        ops[n++] = {"advantages", advantages, 1, rows * 4, 0, false, 4};
        ops[n++] = {"weights", weights, 1, rows * 4, 0, false, 4};
        if (ref_logp) ops[n++] = {"ref_logp", ref_logp, 1, rows * 4, 0, false, 4};
    }
    const size_t without_totals = n;
    if (totals) ops[n++] = {"totals", totals, 1, 16, 0, true, 4};
    rc = check_operands(dev, what, ops, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    const Kernel k = kernel_of<kPolicy>(desc->dtype, static_cast<unsigned int>(desc->vocab), 2 * rows * desc->vocab * es > kStreamBeyond);
    rc = check_grid(dev, what, rows, k.threads);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    if (rows == 0) return totals ? custos_hip_clear(dev, totals, 16) : CUSTOS_HIP_OK;
    RowArgs a;
    std::memset(&a, 0, sizeof a);  // (padding included: recordings compare the arguments of their launches byte by byte)
    a.logits = reinterpret_cast<const void*>(logits);
    a.labels = reinterpret_cast<const int*>(labels);
    a.old_logp = reinterpret_cast<const float*>(old_logp);
    a.ref_logp = reinterpret_cast<const float*>(ref_logp);
    a.advantages = reinterpret_cast<const float*>(advantages);
    a.weights = reinterpret_cast<const float*>(weights);
    a.grad = reinterpret_cast<void*>(logits_grad);
    a.logp = reinterpret_cast<float*>(logp);
    a.pitch = desc->pitch;
    a.grad_pitch = desc->grad_pitch;
    a.vocab = static_cast<unsigned int>(desc->vocab);
    a.inv_t = 1.0 / desc->temperature;
    a.scale2 = static_cast<float>(1.4426950408889634 / desc->temperature);
    a.clip_low = desc->clip_low;
    a.clip_high = desc->clip_high;
    a.kl_coef = desc->kl_coef;
    a.grad_factor = desc->grad_scale / desc->temperature;
    Access acc[9];
    size_t n_acc = 0;
    for (size_t i = 0; i < without_totals; i++) acc[n_acc++] = ops[i].access();
    uint64_t area = 0;
    // (the rows' parts, and behind them the sums of 8192 of them each, and so on)
    const size_t area_bytes = (rows + rows / (kRowsEach / 2) + 64) * sizeof(float4);
    if (totals) {
        rc = operator_workspace(dev, area_bytes, &area);
        if (rc != CUSTOS_HIP_OK) return rc;
        a.terms = reinterpret_cast<float4*>(area);
        acc[n_acc++] = {area, area + rows * sizeof(float4), true};
    }
    const OpArg arg{&a, sizeof a};
    rc = launch(dev, "custos_policy_rows", k.fn, rows, k.threads, &arg, 1, acc, n_acc);
    if (rc != CUSTOS_HIP_OK || !totals) return rc;
    return launch_totals(dev, area, rows, totals);
}

}  // extern "C"
