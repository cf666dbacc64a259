// Host-only tests (no GPU) of the group norm's plans: over many sizes, what the kernels take for granted of a plan.
#include "check.hpp"
#include "../../custos_amd/csrc/group_norm_plan.hpp"

using namespace custos_hip;
using namespace custos_hip::group_norm;

namespace {

custos_hip_group_norm_desc desc_of(int32_t dtype, u64 samples, u64 positions, u64 channels, u64 groups, int32_t flags) {
    return {dtype, CUSTOS_HIP_F32, CUSTOS_HIP_ACT_NONE, flags, samples, positions, channels, groups, 1e-5};
}

// Rows that the parts of a sample stand for, counted part by part as the kernels do.
u64 rows_of(const Splits& s, unsigned int step, u64 positions) {
    u64 rows = 0;
    for (u64 part = 0; part < s.count; part++) {
        const u64 rounds = s.rounds + (part < s.longer ? 1 : 0);
        for (u64 r0 = 0; r0 < step; r0++) {
            u64 mine = rounds;
            const u64 p = part * step + r0;
            if (mine > 0 && p + (mine - 1) * static_cast<u64>(s.count) * step >= positions) mine--;
            rows += mine;
        }
    }
    return rows;
}

// What a kernel reads and writes stays within its shared arrays, and every value belongs to one thread.
bool holds(const Plan& p, const custos_hip_group_norm_desc& d, bool count_rows) {
    const GroupNormArgs& a = p.a;
    const u64 full = 16 / elem_size(d.dtype), width = static_cast<u64>(a.tile_groups) * a.per_group;
    bool ok = a.tile_groups >= 1 && static_cast<u64>(a.tile_groups) * a.tiles == d.groups && a.per_group * d.groups == d.channels;
    ok = ok && (p.vec == 1 || (static_cast<u64>(p.vec) == full && width >= full)) && a.vecs == (width + p.vec - 1) / p.vec && a.step >= 1;
    if (p.in_registers) {
        // tables of threads * vec channels, kMaxTileGroups groups; a thread holds `held` rows of one column
        return ok && a.tile_groups <= kMaxTileGroups && static_cast<u64>(a.step) * a.vecs <= static_cast<u64>(p.threads) &&
               static_cast<u64>(a.step) * p.held >= d.positions && a.parts.count == 1;
    }
    // tables of kBlock * vec channels, kMaxStreamGroups groups; more than one column to a thread only if they are one group's
    ok = ok && a.tile_groups <= static_cast<unsigned int>(kMaxStreamGroups) && (a.tile_groups == 1 || static_cast<u64>(a.step) * a.vecs <= static_cast<u64>(kBlock));
    ok = ok && (a.vecs > static_cast<unsigned int>(kBlock) ? a.step == 1 : static_cast<u64>(a.step) * a.vecs <= static_cast<u64>(kBlock));
    ok = ok && a.parts.count >= 1 && a.values.count >= 1 && static_cast<u64>(a.parts.count) * a.tile_groups <= std::max<u64>(4096, a.tile_groups);
    if (!ok || !count_rows) return ok;
    Plan narrow = p;
    narrow_values(&narrow);
    return rows_of(a.parts, a.part_step, d.positions) == d.positions && rows_of(a.values, a.step, d.positions) == d.positions &&
           rows_of(narrow.a.values, narrow.a.step, d.positions) == d.positions;
}

int plans = 0, streamed = 0;

void check_all(const custos_hip_group_norm_desc& d, bool count_rows) {
    for (int which = 0; which < 3; which++) {
        const Plan p = which == 0 ? forward_plan(d) : gradient_plan(d, which == 2);
        plans++;
        streamed += !p.in_registers;
        if (holds(p, d, count_rows) && fits(p)) continue;
        std::ostringstream o;
        o << (which == 0 ? "forward" : which == 1 ? "gradient" : "gradient from a checkpoint") << (d.flags ? ", stored" : "") << ", "
          << elem_size(d.dtype) << "-byte elements, " << d.samples << "x" << d.positions << "x" << d.channels << " in " << d.groups << " groups: "
          << p.a.tile_groups << " groups and " << p.a.vecs << " vectors a tile, " << p.a.step << " rows" << (p.in_registers ? ", in registers" : "");
        if (check::failures() < 10) check::fail(__FILE__, __LINE__, o.str());
        else check::failures()++;
    }
}

}  // namespace

// Every number of groups against every number of channels in one: in the caches and (third size) beyond 64 MiB.
TEST_CASE(plans_of_all_groupings) {
    for (int32_t dtype : {CUSTOS_HIP_F32, CUSTOS_HIP_BF16})
        for (u64 groups = 1; groups <= 400; groups++)
            for (u64 per_group = 1; per_group <= 300; per_group++) {
                const u64 channels = groups * per_group;
                for (u64 positions : {u64(300), u64(700), (48ull << 20) / channels + 1}) check_all(desc_of(dtype, 1, positions, channels, groups, 0), false);
            }
    CHECK(streamed > plans / 4);
}

TEST_CASE(plans_of_wide_groups_and_large_primes) {
    for (int32_t dtype : {CUSTOS_HIP_F32, CUSTOS_HIP_F16})
        for (u64 groups : {1ull, 2ull, 3ull, 17ull, 127ull, 131ull, 509ull, 1021ull, 2039ull, 4093ull, 8191ull, 2ull * 4093, 127ull * 131})
            for (u64 per_group : {1ull, 3ull, 7ull, 8ull, 15ull, 16ull, 31ull, 33ull, 63ull, 127ull, 129ull, 255ull, 1000ull, 1024ull, 2047ull, 4100ull, 70001ull})
                for (u64 positions : {1ull, 2ull, 40ull, 1000ull, 30000ull})
                    for (u64 samples : {1ull, 3ull, 600ull})
                        for (int32_t flags : {0, CUSTOS_HIP_GRAD_OVERWRITE}) check_all(desc_of(dtype, samples, positions, groups * per_group, groups, flags), false);
}

// Every position belongs to one part, whatever the rounds come to.
TEST_CASE(parts_cover_every_position) {
    for (int32_t dtype : {CUSTOS_HIP_F32, CUSTOS_HIP_BF16})
        for (u64 groups : {1ull, 5ull, 32ull, 37ull, 41ull, 53ull})
            for (u64 per_group : {1ull, 9ull, 31ull, 40ull, 300ull})
                for (u64 samples : {1ull, 2ull, 19ull, 1500ull})
                    for (u64 positions : {1ull, 2ull, 3ull, 255ull, 256ull, 1961ull, 4100ull, 20000ull, 100003ull})
                        check_all(desc_of(dtype, samples, positions, groups * per_group, groups, 0), true);
}

int main(int argc, char** argv) { return check::run(argc, argv); }
