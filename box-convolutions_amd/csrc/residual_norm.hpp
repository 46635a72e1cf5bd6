// How residual_norm.hip deals rows to workgroups.
#pragma once

#include <algorithm>

#include "operators_host.hpp"

namespace boxconv {

namespace {

// The sums over rows that a workgroup of the backward keeps per channel, and where their totals go.
constexpr int kSums = 5, kSumGate = 4;
struct RowGrads { void* p[kSums]; };       // after_weight, after_bias, before_weight, before_bias, gate

// Items (what shares a gate: a batch item, or everything) over workgroups: `parts` workgroups an item with `rows` rows each, or `items` whole
// items a workgroup.
struct RowPlan { int64_t batch, parts, items, rows, groups; };

// About `target` workgroups, of at least `least` rows each where an item is cut.
RowPlan plan_rows(const ResidualNormCall& c, int64_t target, int64_t least) {
    RowPlan p = {1, 1, 1, 0, 0};
    int64_t pixels = c.batch * c.pixels;
    if (c.gate_kind == kGateItem) {
        p.batch = c.batch;
        pixels = c.pixels;
    }
    if (p.batch >= target) {
        p.items = (p.batch + target - 1) / target;
        p.rows = pixels;
        p.groups = (p.batch + p.items - 1) / p.items;
    } else {
        p.parts = std::max<int64_t>(1, std::min(target / p.batch, (pixels + least - 1) / least));
        p.rows = (pixels + p.parts - 1) / p.parts;
        p.parts = (pixels + p.rows - 1) / p.rows;
        p.groups = p.batch * p.parts;
    }
    return p;
}

// Workgroups to aim for in the backward, each of which takes `at_once` rows of an item at a time: those that the chip holds, several times that where a sum over rows would be
// a chain of more than some 256 additions (at most twice that, where items and parts do not divide), whose roundings add up: 2097152 items of one row of 8,
// the same gradient 1.1 everywhere, were off by 4.1e-5 of the sum with 512 workgroups. A grid holds 2^20 workgroups of up to 1024 threads.
int64_t backward_target(const ResidualNormCall& c, int64_t at_once, int64_t resident) {
    const int64_t items = c.gate_kind == kGateItem ? c.batch : 1, pixels = c.gate_kind == kGateItem ? c.pixels : c.batch * c.pixels;
    const int64_t wanted = std::min<int64_t>(int64_t(1) << 20, (items * ((pixels + at_once - 1) / at_once) + 255) / 256);
    return std::max<int64_t>(1, (wanted + resident - 1) / resident) * resident;        // (whole rounds of them: 300007 items of 40 channels 1.7 ms, 2.2 otherwise)
}

// Items of a workgroup. (The last ones have fewer, where they do not divide: what is read by an item's number has to stop with them.)
__host__ __device__ inline int64_t items_of(const RowPlan& p, int64_t group) {
    const int64_t left = p.batch - group * p.items;
    return p.parts > 1 ? 1 : left < p.items ? left : p.items;
}

// The rows [first, last) of item i of the workgroup's items_of, counted over the whole tensor.
struct Span { int64_t item, first, last; };
__host__ __device__ inline Span span_of(const RowPlan& p, int64_t pixels, int64_t group, int64_t i) {
    const int64_t item = p.parts > 1 ? group / p.parts : group * p.items + i, begin = p.parts > 1 ? group % p.parts * p.rows : 0;
    const int64_t end = begin + p.rows < pixels ? begin + p.rows : pixels;
    return {item, item * pixels + begin, item * pixels + end};
}

}  // namespace

}  // namespace boxconv
