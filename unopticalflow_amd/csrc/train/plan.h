// Which tile size a launch takes, and into how many shares its sums are cut, from a model of what the launch costs.
//
// A launch works on jobs: `tiles` tiles of a side, each summing over `stages` stages of 64 packed elements.  A tile of side 256 has the best rate
// (an operand is read once for 256 rows of the other), smaller ones fill the chip better; sums cut into shares fill it too, but leave fp32
// partial sums that are written, read and added.  The model: units (a share of a tile) run on `slots` places in rounds of the longest
// unit; a unit costs its stages times the measured time of one, and a start and an end.
#pragma once
#include "mfma16.h"
#include <cmath>

namespace {

constexpr int kVariants = 6;
// of the variants of with_tile(): the last two with more stages in LDS, fewer on a CU
constexpr int kSizes[kVariants] = {256, 192, 128, 64, 128, 64};

// m x n outputs (lower: the lower triangle of m x m) of `times` matrices, `out` bytes written for each; cut: may be cut into shares
struct Job { long long m, n; int stages; bool lower, cut; double out; int times = 1; };
struct Choice { int size, limit; double us; };                            // index into kSizes; stages of the longest share

// how many shares a sum of `stages` is cut into so that none is longer than `limit` (at most 16 shares, none empty)
static int shares_of(int stages, int limit) {
    int shares = (stages + limit - 1) / limit;
    shares = shares > 16 ? 16 : shares < 1 ? 1 : shares;
    const int each = (stages + shares - 1) / shares;
    return each > 0 ? (stages + each - 1) / each : 1;
}
static int stages_of(long long packed_width_) { return (int)((packed_width_ + 63) / 64); }

static long long tiles_of(long long m, long long n, int size) { return ((m + size - 1) / size) * ((n + size - 1) / size); }
static long long lower_tiles_of(long long m, int size) { const long long t = (m + size - 1) / size; return t * (t + 1) / 2; }

// Measured: microseconds of one stage of a unit on a full chip (of the units that share a CU, together) and on an empty one (a chip is as slow as a
// full one from 60 % on), and of a unit's start and end.  (8192 x 8192 x 2048 against x 512, and 1024 x 1024 x 4096; ONE and TWO planes)
struct Cost { double full, alone, ends; int per_cu; };
static const Cost kCost[2][kVariants] = {
    {{1.50, 1.10, 10., 1}, {0.97, 0.68, 7., 1}, {1.10, 0.62, 5., 2}, {0.80, 0.46, 4., 4}, {0.53, 0.45, 5., 1}, {0.35, 0.26, 4., 2}},
    {{2.15, 1.50, 18., 1}, {1.28, 0.95, 11., 1}, {1.25, 0.60, 7.5, 2}, {0.83, 0.44, 4.8, 4}, {0.64, 0.54, 7.5, 1}, {0.44, 0.28, 4.5, 2}}};
constexpr double kJoinBytesPerUs = 3.0e6, kLaunchUs = 5.0, kStoreBytesPerUs = 4.5e6 / 256.;          // joining: the chip; stores: a CU's part of it

static Choice choose(int planes, const Job* jobs, int count) {
    Choice best{0, 1, -1.};
    int longest = 1;
    bool any = false;
    for (int i = 0; i < count; ++i) {
        if (jobs[i].cut && jobs[i].stages > longest) longest = jobs[i].stages;
        any = any || jobs[i].cut;
    }
    for (int z = 0; z < kVariants; ++z) {
        const Cost& c = kCost[planes == TWO ? 1 : 0][z];
        for (int s = 1; s <= 16; s = s < 4 ? s + 1 : s < 8 ? s + 2 : s + 4) {
            const int limit = (longest + s - 1) / s;
            if (s > 1 && (!any || limit < 4)) break;
            int most = 0, least = 1 << 30;                                 // stages of a unit
            double sum = 0., joined = 0., all = 0., longest_us = 0., least_us = 1e30, ends = 0.;
            for (int i = 0; i < count; ++i) {
                const int shares = jobs[i].cut ? shares_of(jobs[i].stages, limit) : 1, each = (jobs[i].stages + shares - 1) / shares;
                const double units = (double)jobs[i].times * (jobs[i].lower ? lower_tiles_of(jobs[i].m, kSizes[z]) : tiles_of(jobs[i].m, jobs[i].n,
                    kSizes[z])) * shares;
                const double area = (double)kSizes[z] * kSizes[z],
                    end = c.ends + c.per_cu * area * (shares > 1 ? 4. : jobs[i].out) / kStoreBytesPerUs, us = each * c.full + end;
                if (us > longest_us) { longest_us = us; most = each; ends = end; }
                least = each < least ? each : least;
                least_us = us < least_us ? us : least_us;
                sum += units * us;
                all += units;
                if (shares > 1) joined += units * area * 8.;
            }
            const double slots = 256. * c.per_cu, units = sum / longest_us;          // (in units of the longest)
            if (z >= 4 && all > slots) break;                              // many stages in LDS only serve what runs at once
            auto last = [&](double n) {                                    // the longest unit among n that run together, n <= slots
                const double busy = 1.6 * n / slots, part = busy < 1. ? busy : 1.;
                return most * (c.alone + (c.full - c.alone) * part) + c.ends + (ends - c.ends) * part;
            };
            double us;
            if (units <= slots) us = last(units);
            else if (least == most) {
                const double rounds = floor(units / slots), rest = units - rounds * slots;
                us = rounds * longest_us + (rest > 0.5 ? last(rest) : 0.);
            } else us = units / slots * longest_us + 0.5 * least_us;                                     // the short ones fill up
            us += joined > 0. ? kLaunchUs + joined / kJoinBytesPerUs : 0.;
            if (best.us < 0. || us < best.us) best = Choice{z, limit, us};
        }
    }
    return best;
}

}  // namespace
