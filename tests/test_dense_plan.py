"""Cuts and workspaces of the dense layers, over many sizes and without a GPU: the header that lays them out is plain C++.

A call may ask for any of its gradients ("each output may be NULL").  Whatever it asks for, the sums of a cut contraction, the copies
and the column sums have to fit what v2vae_linear_workspace_bytes and v2vae_gated_workspace_bytes said."""
import os
import subprocess

import pytest

from volterra_vae_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdio>
#include "v2vae_dense_plan.h"
using namespace v2vae;

static long long sizes = 0, cut = 0, beyond = 0;
static void fits(const v2vae_dense& d, bool gated, const char* what, size_t need, size_t room) {
    cut += need > 0;
    if (need <= room) return;
    if (beyond++ < 20)
        std::printf("beyond: dtype %d gated %d %lld x %lld -> %lld (ld_x %lld) %s: %zu of %zu\n", d.dtype, gated, (long long)d.rows,
                    (long long)d.in, (long long)d.out, (long long)d.ld_x, what, need, room);
}
// every cut, either alignment; `formed` of a product's batch entries are written
static void product(const v2vae_dense& d, bool gated, const char* what, const Product& p, int formed, size_t room) {
    for (int direct = 0; direct < (d.dtype == V2VAE_F32 ? 1 : 2); ++direct) {
        const Cut c = cut_product(p, d.dtype, direct);
        const int64_t step = d.dtype == V2VAE_F32 ? 32 : 64, steps = (p.K + step - 1) / step * p.segs;
        if ((int64_t)c.splits * c.per < steps || (int64_t)(c.splits - 1) * c.per >= (steps > 0 ? steps : 1)) {
            std::printf("beyond: parts of %s\n", what);
            ++beyond;
        }
        fits(d, gated, what, c.splits > 1 ? (size_t)c.splits * formed * p.M * p.N * (p.gated ? 2 : 1) * 4 : 0, room);
    }
}
int main() {
    const int64_t rows[] = {0, 1, 16, 17, 33, 64, 100, 300, 500, 512, 1000, 1024, 2048, 3000, 4096, 4999, 10000, 32768, 65536, 262144};
    const int64_t widths[] = {1, 7, 25, 50, 64, 96, 130, 250, 256, 300, 512, 515, 700, 1000, 1024, 1280, 2000, 2048, 2560, 4095, 4096, 5632};
    for (int dtype = V2VAE_F32; dtype <= V2VAE_F16; ++dtype)
        for (int gated = 0; gated < 2; ++gated)
            for (int act = 0; act < 2; ++act)
                for (int pad = 0; pad < 2; ++pad)
                    for (int64_t m : rows)
                        for (int64_t k : widths)
                            for (int64_t n : widths) {
                                const v2vae_dense d = {dtype, act, m, k, n, k + pad, k, k + 3 * pad, n, n + pad};
                                if (check_dense(&d, gated, true, true) != V2VAE_OK) continue;
                                ++sizes;
                                if (m > few_rows(dtype)) {
                                    const FwdLayout f = fwd_layout(&d, gated);
                                    product(d, gated, "y", forward_product(&d, gated), 1, f.total - f.prod);
                                    fits(d, gated, "copies", planes_of(&d, gated, false).bytes + packs_of(&d, gated, false).x_bytes +
                                                                 packs_of(&d, gated, false).w_bytes, f.prod);
                                }
                                const BwdLayout b = bwd_layout(&d, gated);
                                product(d, gated, "dx", input_product(&d, gated), 1, b.total - b.prod);
                                for (int formed = 1; formed <= 1 + gated; ++formed)
                                    product(d, gated, formed == 1 ? "one dw" : "both dw", weight_product(&d, gated), formed, b.total - b.prod);
                                const Packs p = packs_of(&d, gated, true);
                                if (gated || act || p.dz)
                                    for (int q = 0; q <= gated; ++q)
                                        fits(d, gated, "dz", (size_t)m * p.ld_out * elem_bytes(dtype), (q < gated ? b.dz[1] : b.part[0]) - b.dz[q]);
                                for (int64_t width : {n, (int64_t)p.ld_out}) {
                                    int cx, gx, chunks;
                                    slope_shape(m, width, &cx, &gx, &chunks);
                                    for (int q = 0; q <= gated; ++q)
                                        fits(d, gated, "column sums", (size_t)chunks * n * 4, (q < gated ? b.part[1] : b.planes) - b.part[q]);
                                }
                                fits(d, gated, "planes", planes_of(&d, gated, true).bytes, b.x - b.planes);
                                fits(d, gated, "copy of x", p.x_bytes, b.w - b.x);
                                fits(d, gated, "copy of w", p.w_bytes, b.prod - b.w);
                            }
    const v2vae_dense some[] = {SOME};
    for (const v2vae_dense& d : some)
        std::printf("bytes %zu %zu %zu %zu\n", fwd_layout(&d, false).total, bwd_layout(&d, false).total, fwd_layout(&d, true).total,
                    bwd_layout(&d, true).total);
    std::printf("sizes %lld cut %lld beyond %lld\n", sizes, cut, beyond);
    return beyond != 0;
}
"""
SOME = [(dtype, act, m, k, n, k, k, k, n, n) for dtype in range(3) for act in (0, 2)
        for m, k, n in ((5, 9000, 40), (300, 2000, 256), (1024, 2048, 512), (4096, 2048, 1000), (4001, 2047, 515), (500, 1024, 256))]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    here = tmp_path_factory.mktemp("plan")
    source, binary = here / "plan.cpp", here / "plan"
    source.write_text(PROGRAM.replace("SOME", ", ".join("{%s}" % ", ".join(map(str, s)) for s in SOME)))
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "volterra_vae_amd", "csrc"), "-o", str(binary),
                    str(source)], check=True)
    return subprocess.run([str(binary)], capture_output=True, text=True, timeout=300)


def test_every_cut_of_every_choice_of_gradients_fits_its_workspace(plan):
    sizes, cut, beyond = (int(v) for v in plan.stdout.splitlines()[-1].split()[1::2])
    assert sizes > 100000 and cut > 100000, plan.stdout
    assert beyond == 0 and plan.returncode == 0, plan.stdout


def test_the_library_reports_these_workspaces(plan):
    reported = [tuple(int(v) for v in line.split()[1:]) for line in plan.stdout.splitlines() if line.startswith("bytes")]
    lin, gat = _lib.lib.v2vae_linear_workspace_bytes, _lib.lib.v2vae_gated_workspace_bytes
    for s, r in zip(SOME, reported, strict=True):
        d = _lib.Dense(*s)
        assert (lin(d, 0), lin(d, 1), gat(d, 0), gat(d, 1)) == r
