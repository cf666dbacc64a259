// Plans of the group norm's launches: which tile of the data a workgroup takes, and how the positions of a sample are
// dealt out (group_norm.hip).  Host code only.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <utility>

#include "../../include/custos_hip.h"

namespace custos_hip {

typedef unsigned long long u64;

namespace group_norm {

constexpr int kBlock = 256;      // threads of the kernels that stream
constexpr unsigned int kMaxTileGroups = 64;     // groups per tile of the kernels that hold a tile in registers
constexpr int kAheadForward = 4, kAheadBackward = 2;  // rows a thread of the kernels that stream loads before it uses them
constexpr int kMaxStreamGroups = 128;  // groups per tile of the kernels that stream

// Division of 32-bit numbers by one the host knows.
struct Divisor {
    unsigned int by, magic;  // floor(2^32 / by); by == 1: 0, and the correction below gives the answer
};
// How the rows of a sample are dealt out to workgroups: `rounds` rounds of `step` rows each, to the first `longer` of
// them one more.
struct Splits {
    unsigned int count, longer;
    u64 rounds;
    Divisor by_count;
};

struct GroupNormArgs {
    const void* x;            // or null: codes and scales of an 8-bit checkpoint
    const signed char* codes;
    const float* scales;
    const void* gamma;        // null: ones
    const void* beta;         // null: zeros
    const void* out_grad;     // backward
    void* out;                // out, or x_grad
    float* stats;             // [samples][groups]: mean, rstd
    // Work area, a "part" being the positions of a sample that one workgroup of the first pass takes (all of them for
    // a tile in registers).  Forward: [samples][parts][groups] pairs of a mean and a sum of squared
    // distances.  Backward: the same of the sums of dz * gamma and of dz * gamma * h, and `channel_parts`.
    float* group_parts;
    float* channel_parts;     // [channel_rows][2][channels]: sums of dz and of dz * h
    float* gamma_grad;
    float* beta_grad;
    u64 positions;
    u64 x_pitch, grad_pitch, out_pitch;
    unsigned int samples, channels, groups, per_group, tile_groups, tiles;
    Splits parts, values;          // of the first pass (a part each), and of the second
    Divisor by_tiles;
    unsigned int vecs, vecs_magic; // vectors per row of a tile; ceil(2^32 / vecs)
    unsigned int waves_per_group, waves_magic;  // where a tile has fewer groups than a workgroup has wavefronts
    double total_inverse;          // 1 / values of a group
    int whole_groups;              // no vector of a row has channels of two groups
    unsigned int step;             // rows a workgroup of a streaming kernel reads at a time
    unsigned int part_step;        // the first pass's
    unsigned int last_part, missing_rows;  // the part with the last round of rows, and how many that is short of `step`
    unsigned int blocks;           // workgroups that work on values; what follows them adds up gamma_grad and beta_grad
    unsigned int channel_rows;     // of channel_parts: a part each, or the samples that one workgroup takes
    unsigned int per_group_magic;  // ceil(2^32 / per_group), for divisions of numbers below 2^16
    int param_f32, accumulate;
    float eps;
};

// What the plans below go by, in microseconds measured on MI355X (kernels alone):
// - Rows of a tile in registers are at least 32 bytes: twice the workgroups of 64-byte rows, 8x1024x640 bf16 in
//   12.8 against 14.6 (41 with 128 bytes); the tiles that share a cache line run on one XCD.
//   Wider ones while 256 threads hold them with four vectors each and 1024 tiles are left: every workgroup waits for
//   the same few loads and barriers, however little it moves.  512x64x640 bf16 in 26 forward and 71 backward, against 56
//   and 150 with rows of 32 bytes; 64x64x1280 in 11 and 20 against 15 and 28.
// - Rows of a tile that is streamed are at least 128 bytes: the second pass of the gradient over 4x4096x320 bf16
//   takes 10.9, with 256 bytes 12.2, with 64 bytes 15.2; the first pass 11.8, 11.4, 13.7.  Where the data does not
//   stay in the caches, 256 bytes: gradient over 8x16384x512 bf16 from codes 49 + 57, with 128 bytes 50 + 79, with
//   512 bytes 48 + 60.
// - A tile of more than 16384 values is only held if there are at least 128 of them: 33 tiles of 58830 f32 values
//   with GELU take 28 on 33 of 256 CUs, two streaming passes over the same data 16.
// - Beyond 64 MiB moved the second pass loads and stores past the caches: its results would only push out what the
//   first pass read and leave dirty lines to be written back during the next pass.  16x16384x512 f16: first pass
//   55 and second 88 that way, 85 and 102 through the caches.
constexpr unsigned int kTileRow = 32, kStreamRow = 128;
// - Tiles in registers, backward: beyond 2^21 threads, four times what the chip holds at once, a workgroup takes
//   several samples.
constexpr u64 kTilesEnough = 1024;
constexpr u64 kThreadsTogether = 1ull << 21;
constexpr u64 kTileAlone = 16384, kTilesTogether = 128, kStreamBeyond = 64ull << 20;

struct Plan {
    int vec = 1;                // channels per thread
    bool in_registers = false;
    int threads = kBlock;
    int held = 0;
    bool stream = false;  // the second pass loads and stores past the caches
    GroupNormArgs a;
    // (padding included: recordings compare the arguments of their launches byte by byte)
    Plan() { std::memset(&a, 0, sizeof a); }
};

inline Divisor divisor(unsigned int by) { return {by, by == 1 ? 0u : static_cast<unsigned int>(0x100000000ull / by)}; }

inline unsigned int magic_of(unsigned int d) { return d == 1 ? 0u : static_cast<unsigned int>((0x100000000ull + d - 1) / d); }

// The smallest divisor of `groups` whose tile is at least `channels` wide (or all groups); if it is above `most`, or its
// tile wider than `widest`, the largest one below (at the least one group, however wide).
inline unsigned int tile_at_least(unsigned int groups, unsigned int per_group, unsigned int channels, unsigned int most, u64 widest) {
    unsigned int best = 1;
    for (unsigned int k = 1; k <= std::min(groups, most); k++)
        if (groups % k == 0) {
            if (k > 1 && static_cast<u64>(k) * per_group > widest) break;
            best = k;
            if (static_cast<u64>(k) * per_group >= channels) break;
        }
    return best;
}
// (threads, vectors held) of the kernels that hold a tile in registers, smallest first, and the most bytes moved they
// are used for: one reading of x in rows of 32 bytes against two readings in wide ones, the second of which finds x
// in the caches.  Forward, 1024 x 8: 8x4096x512 bf16 (64 MiB) in 22 against 27 streamed, 16x4096x512 in 49 against 41;
// 1024 x 16: 4x4096x640 bf16 (40 MiB) in 23 against 26, 4x4096x512 f32 in 20 against 24, but 4x7000x512 bf16 in 29
// against 26.  Backward, 512 x 4: 4x256x1280 bf16 (7.5 MiB) in 12 against 20, 8x256x1280 in 13 against 20, 8x1024x320
// in 19 both ways, 16x512x1024 (48 MiB) in 27 against 24; 1024 threads leave that kernel too few registers.
struct Held {
    int threads, held;
    u64 most;
};
constexpr Held kForwardHeld[] = {{256, 4, ~0ull}, {256, 8, ~0ull}, {1024, 4, ~0ull}, {1024, 8, kStreamBeyond}, {1024, 16, kStreamBeyond}};
constexpr Held kBackwardHeld[] = {{256, 4, ~0ull}, {512, 4, 32ull << 20}};

// `accumulates`: the results are added to what is there, so no channel may be stored by two threads.  `rounds_each`: the
// fewest rounds of rows of a workgroup of the first pass.
template <size_t N>
void make_plan(const custos_hip_group_norm_desc& d, size_t elem, u64 moved, bool accumulates, const Held (&choices)[N], u64 rounds_each, Plan* plan) {
    GroupNormArgs& a = plan->a;
    a.positions = d.positions;
    a.samples = static_cast<unsigned int>(d.samples);
    a.channels = static_cast<unsigned int>(d.channels);
    a.groups = static_cast<unsigned int>(d.groups);
    a.per_group = a.channels / a.groups;
    a.per_group_magic = magic_of(a.per_group);
    a.eps = static_cast<float>(d.eps);
    const unsigned int full = static_cast<unsigned int>(16 / elem);
    auto finish = [&](u64 parts, u64 values) {
        a.part_step = a.step;
        const u64 rounds = (a.positions + a.step - 1) / a.step;
        for (auto [of, count] : {std::pair<Splits*, u64>{&a.parts, parts}, std::pair<Splits*, u64>{&a.values, values}}) {
            of->count = static_cast<unsigned int>(count);
            of->rounds = rounds / count;
            of->longer = static_cast<unsigned int>(rounds % count);
            of->by_count = divisor(of->count);
        }
        a.last_part = static_cast<unsigned int>((rounds - 1) % parts);
        a.missing_rows = static_cast<unsigned int>(rounds * a.step - a.positions);
        a.by_tiles = divisor(a.tiles);
        a.vecs_magic = magic_of(a.vecs);
        a.waves_per_group = std::max(1u, static_cast<unsigned int>(plan->threads) / 64 / a.tile_groups);
        a.waves_magic = magic_of(a.waves_per_group);
        a.whole_groups = a.tile_groups == 1 || a.per_group % static_cast<unsigned int>(plan->vec) == 0;
        a.total_inverse = 1.0 / (static_cast<double>(a.positions) * a.per_group);
    };
    // in registers, if a tile of whole groups fits whose rows are at least kTileRow bytes
    {
        unsigned int k = tile_at_least(a.groups, a.per_group, static_cast<unsigned int>(kTileRow / elem), kMaxTileGroups, ~0ull);
        for (unsigned int wider = k + 1; wider <= std::min(a.groups, kMaxTileGroups); wider++) {
            const u64 row = (static_cast<u64>(wider) * a.per_group + full - 1) / full;
            if (row > kBlock || a.positions > 4 * (kBlock / row) || static_cast<u64>(a.samples) * (a.groups / wider) < kTilesEnough) break;
            if (a.groups % wider == 0) k = wider;
        }
        const u64 width = static_cast<u64>(k) * a.per_group;
        const unsigned int vec = width < full || (accumulates && width % full != 0) ? 1 : full;
        const u64 vecs = (width + vec - 1) / vec;
        for (const Held& h : choices) {
            if (vecs > static_cast<u64>(h.threads) || moved > h.most) continue;
            const u64 step = static_cast<u64>(h.threads) / vecs;
            if ((a.positions + step - 1) / step > static_cast<u64>(h.held)) continue;
            if (a.positions * width > kTileAlone && static_cast<u64>(a.samples) * (a.groups / k) < kTilesTogether) continue;
            plan->in_registers = true;
            plan->vec = static_cast<int>(vec);
            plan->threads = h.threads;
            plan->held = h.held;
            a.tile_groups = k;
            a.tiles = a.groups / k;
            a.vecs = static_cast<unsigned int>(vecs);
            a.step = static_cast<unsigned int>(step);
            finish(1, 1);
            return;
        }
    }
    // (of several groups only as wide as one vector a thread: the first pass keeps one column's sums, or one group's.
    // With 17, 37, 41 groups and other primes the next divisor is all of them.)
    a.tile_groups = tile_at_least(a.groups, a.per_group, static_cast<unsigned int>((moved > kStreamBeyond ? 2 * kStreamRow : kStreamRow) / elem), kMaxStreamGroups,
                                  static_cast<u64>(kBlock) * full);
    const u64 width = static_cast<u64>(a.tile_groups) * a.per_group;
    plan->vec = static_cast<int>(width < full ? 1 : full);
    a.tiles = a.groups / a.tile_groups;
    const u64 vecs = (width + plan->vec - 1) / plan->vec;
    a.vecs = static_cast<unsigned int>(vecs);
    a.step = static_cast<unsigned int>(std::max<u64>(1, kBlock / vecs));
    const u64 rounds = (a.positions + a.step - 1) / a.step, tiles = static_cast<u64>(a.samples) * a.tiles;
    plan->stream = moved > kStreamBeyond;
    // What the chip holds at once, each with a few rounds of rows, and no more parts than are joined in passing.  In the
    // first pass two rounds of loads on the way to each thread: 8 rows forward, 4 backward (forward over 3x1961x330 f32
    // 16.0, with 4 rows 17.3, with 2 21; over 20000x64 bf16 14.4, 15.5, 16.0; gradient over 4x1024x640 bf16 18.7, with 8
    // rows 20.5), in the second 4 (with 8 the last two take 16.6 and 20.9).
    finish(std::min<u64>({std::max<u64>(1, 1024 / tiles), std::max<u64>(1, rounds / rounds_each), std::max<u64>(1, 4096 / a.tile_groups)}),
           std::min<u64>(std::max<u64>(1, 2048 / tiles), std::max<u64>(1, rounds / 4)));
}

// What the kernels take for granted: their shared arrays hold a row of every thread, one group per tile or one column per
// thread, and the groups of a tile.
inline bool fits(const Plan& plan) {
    const GroupNormArgs& a = plan.a;
    if (plan.in_registers)
        return a.tile_groups <= kMaxTileGroups && static_cast<u64>(a.step) * a.vecs <= static_cast<u64>(plan.threads) &&
               a.positions <= static_cast<u64>(a.step) * static_cast<u64>(plan.held);
    return a.tile_groups <= static_cast<unsigned int>(kMaxStreamGroups) && (a.tile_groups == 1 || static_cast<u64>(a.step) * a.vecs <= static_cast<u64>(kBlock));
}

// The second pass of a streaming plan whose rows are no whole vectors and whose results are added to, or take the place
// of, what it reads: channel by channel, so that none is stored, or read after it was stored, by another thread.
inline void narrow_values(Plan* plan) {
    GroupNormArgs& a = plan->a;
    if (plan->vec == 1 || a.tile_groups * a.per_group % static_cast<unsigned int>(plan->vec) == 0) return;
    plan->vec = 1;
    a.vecs = a.tile_groups * a.per_group;
    a.vecs_magic = magic_of(a.vecs);
    a.step = std::max(1u, static_cast<unsigned int>(kBlock) / a.vecs);
    a.whole_groups = 1;
    const u64 rounds = (a.positions + a.step - 1) / a.step;
    a.values.count = static_cast<unsigned int>(std::min<u64>(a.values.count, std::max<u64>(1, rounds / 4)));
    a.values.rounds = rounds / a.values.count;
    a.values.longer = static_cast<unsigned int>(rounds % a.values.count);
    a.values.by_count = divisor(a.values.count);
}

inline size_t elem_size(int32_t dtype) { return dtype == CUSTOS_HIP_F32 ? 4 : 2; }

// The plans of both directions, of sizes that check_desc has let pass and that are not empty.  `saved`: x is an 8-bit
// checkpoint.
inline Plan forward_plan(const custos_hip_group_norm_desc& d) {
    Plan plan;
    const size_t es = elem_size(d.dtype);
    make_plan(d, es, 2 * d.samples * d.positions * d.channels * es, /*accumulates=*/false, kForwardHeld, 2 * kAheadForward, &plan);
    return plan;
}
inline Plan gradient_plan(const custos_hip_group_norm_desc& d, bool saved) {
    Plan plan;
    const size_t es = elem_size(d.dtype);
    make_plan(d, es, d.samples * d.positions * d.channels * (saved ? 2 * es + 1 : 3 * es),
              /*accumulates=*/!(d.flags & CUSTOS_HIP_GRAD_OVERWRITE), kBackwardHeld, 2 * kAheadBackward, &plan);
    return plan;
}

}  // namespace group_norm

}  // namespace custos_hip
