"""How ``residual_norm`` deals rows to workgroups (csrc/residual_norm.hpp), walked on the CPU as its kernels walk it: a per-item gate is read by the item's
number, so no workgroup may come to an item that is not there."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "box-convolutions_amd", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "residual_norm.hpp"
using namespace boxconv;

int main() {
    const int64_t batches[] = {1, 2, 3, 7, 127, 128, 129, 255, 256, 257, 511, 513, 600, 700, 1023, 1024, 1025, 1300, 2047, 2049, 2100, 4097, 65537};
    const int64_t targets[] = {128, 256, 512, 768, 1024, 2048, 4096};
    long walked = 0, spare = 0;
    for (const int kind : {kGateNone, kGateChannel, kGateItem, kGateFull})
        for (const int64_t batch : batches)
            for (const int64_t pixels : {1, 2, 3, 31, 1000, 4099})
                for (const int64_t target : targets)
                    for (const int64_t least : {1, 4, 16, 32, 256}) {
                        ResidualNormCall c = {};
                        c.gate_kind = kind;
                        c.batch = batch;
                        c.pixels = pixels;
                        const RowPlan p = plan_rows(c, target, least);
                        const int64_t items = kind == kGateItem ? batch : 1, of_item = kind == kGateItem ? pixels : batch * pixels;
                        const auto complain = [&](const char* what, int64_t group, int64_t item) {
                            printf("%s: kind %d, %lld items of %lld rows, target %lld, least %lld: workgroup %lld of %lld, item %lld\n", what, kind, (long long)batch,
                                   (long long)pixels, (long long)target, (long long)least, (long long)group, (long long)p.groups, (long long)item);
                            return 1;
                        };
                        int64_t next = 0;                                // rows and items come in order, every row once
                        for (int64_t group = 0; group < p.groups; ++group) {
                            const int64_t count = items_of(p, group);
                            if (count < 1 || count > p.items) return complain("no items, or too many", group, count);
                            spare += p.items - count;
                            for (int64_t i = 0; i < count; ++i) {
                                const Span s = span_of(p, of_item, group, i);
                                if (s.item < 0 || s.item >= items) return complain("an item that is not there", group, s.item);
                                if (s.first != next || s.last <= s.first) return complain("rows left out, or none", group, s.item);
                                if (s.first < s.item * of_item || s.last > (s.item + 1) * of_item) return complain("another item's rows", group, s.item);
                                next = s.last;
                                ++walked;
                            }
                        }
                        if (next != batch * pixels) return complain("rows left over", p.groups, -1);
                    }
    printf("%ld spans, %ld places without an item\n", walked, spare);
    return walked > 0 && spare > 0 ? 0 : 1;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    folder = tmp_path_factory.mktemp("row_plan")
    source, program = folder / "walk.cpp", folder / "walk"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include", "-I" + CSRC, str(source), "-o", str(program)], check=True)
    return str(program)


def test_no_workgroup_comes_to_an_item_that_is_not_there(walk):
    done = subprocess.run([walk], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout


def test_kernels_walk_as_the_test_does():
    """Every loop over a workgroup's items in the kernels ends where ``items_of`` says."""
    with open(os.path.join(CSRC, "residual_norm.hip")) as file:
        source = file.read()
    calls = source.count("span_of(")
    assert calls == 4 and source.count("i < items_of(a.plan, blockIdx.x); ++i) {\n        const Span span = span_of(a.plan, a.pixels, blockIdx.x, i);") == calls


CHAINS = r"""
#include <cstdio>
#include "residual_norm.hpp"
using namespace boxconv;

int main() {
    long most = 0;
    for (const int kind : {kGateChannel, kGateItem})
        for (int64_t batch = 1; batch < 100000000; batch = batch * 3 + 1)
            for (int64_t pixels = 1; pixels < 100000000 && batch * pixels < 10000000000; pixels = pixels * 5 + 2)
                for (const int64_t at_once : {1, 4, 32, 256})
                    for (const int64_t resident : {128, 256, 512, 1024}) {
                        ResidualNormCall c = {};
                        c.gate_kind = kind;
                        c.batch = batch;
                        c.pixels = pixels;
                        const RowPlan p = plan_rows(c, backward_target(c, at_once, resident), at_once);
                        const int64_t chain = p.items * ((p.rows + at_once - 1) / at_once);        // rows that one team adds up
                        const bool large = batch * pixels / at_once > int64_t(1) << 28;             // (more rows than a GPU's memory holds)
                        if (chain > most && !large) most = chain;
                        if ((chain > 512 && !large) || p.groups >= (int64_t(1) << 32) / 512) {
                            printf("%lld items of %lld rows, %lld at once, %lld workgroups resident: %lld workgroups, a chain of %lld\n", (long long)batch, (long long)pixels,
                                   (long long)at_once, (long long)resident, (long long)p.groups, (long long)chain);
                            return 1;
                        }
                    }
    printf("chains of at most %ld\n", most);
    return most > 1 ? 0 : 1;
}
"""


def test_sums_over_rows_are_short_chains(tmp_path):
    """However many rows and items there are, a team of lanes adds few of them up one after the other."""
    source, program = tmp_path / "chains.cpp", tmp_path / "chains"
    source.write_text(CHAINS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include", "-I" + CSRC, str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout
