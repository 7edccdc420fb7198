"""inzg_expert_lists on devices that cannot hold a cluster of sixteen blocks: the same lists from eight blocks and from one, whichever the
context found possible when it was made. Built from the kernel's source, since this GPU holds sixteen."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "inferenz_b200", "csrc")

SOURCE = """
#include "k_lists.cu"
extern "C" {
int most_cluster(int sixteen, int eight) { return inzg::lists_most_cluster(sixteen, eight); }
int found() { return inzg::lists_set_attributes(); }
int run(int n, int topk, int E, void *sel, void *w, void *off, void *rows, void *slots, void *w_out, int most, void *err) {
    inzg::launch_expert_lists(n, topk, E, (int32_t *)sel, (float *)w, (int32_t *)off, (int32_t *)rows, (int32_t *)slots, (float *)w_out, most,
                              (int32_t *)err, nullptr);
    return (int)cudaGetLastError();
}
}
"""


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("lists")
    (d / "lists.cu").write_text(SOURCE)
    so = str(d / "lists.so")
    subprocess.run([nvcc, "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
                    "--expt-relaxed-constexpr", "-I", CSRC, "-I", os.path.join(ROOT, "include"), str(d / "lists.cu"), "-o", so], check=True)
    return ctypes.CDLL(so)


def test_the_largest_cluster_that_is_possible(built):
    assert [built.most_cluster(*a) for a in ((1, 1), (1, 0), (0, 1), (0, 0))] == [16, 16, 8, 1]


@pytest.mark.gpu
def test_lists_of_every_cluster_size(built):
    import torch
    assert built.found() in (16, 8, 1)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for n, K, E in [(4096, 10, 512), (1000, 16, 2048), (2049, 1, 7), (20_000, 10, 512), (300, 9, 33)]:
        g = torch.Generator(device="cuda").manual_seed(n)
        sel = torch.randint(-E // 3, E, (n, K), generator=g, device="cuda").to(torch.int32)
        w = torch.rand(n, K, generator=g, device="cuda")
        flat = sel.reshape(-1).cpu().numpy().astype(np.int64)
        key = np.where(flat < 0, E, flat)
        order = np.argsort(key, kind="stable")
        order = order[key[order] < E]
        for most in {built.found(), 8, 1} if built.found() > 1 else {1}:
            off = torch.full((E + 1,), -5, dtype=torch.int32, device="cuda")
            rows, slots = (torch.full((n * K,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
            wo, err = torch.full((n * K,), -7.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            assert built.run(n, K, E, p(sel), p(w), p(off), p(rows), p(slots), p(wo), most, p(err)) == 0
            torch.cuda.synchronize()
            m = len(order)
            assert np.array_equal(off.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]))
            assert np.array_equal(slots.cpu().numpy()[:m], order) and np.array_equal(rows.cpu().numpy()[:m], order // K)
            assert torch.equal(wo[:m], w.reshape(-1)[slots[:m].long()]) and bool((slots[m:] == -7).all()) and int(err) == 0
