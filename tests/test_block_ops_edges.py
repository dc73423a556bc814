"""The transformer-block operators at their edges: values far apart, rows that
are not finite, clusters, lanes longer than their hints, buffers in host
memory. Tolerances as in test_block_ops, unless a test derives its own."""

from __future__ import annotations

import math
from pathlib import Path

import pytest
import torch

from ppocr_native_b200 import cuda
from test_block_ops import DTYPES, Q4, Attn, half_step, norm_check

gpu = pytest.mark.gpu
CSRC = Path(cuda.__file__).resolve().parent / "csrc"


# ---------------------------------------------------------------- the 4-bit product

def test_q4_clusters_have_started_before_remote_stores():
    # a block may write into another's shared memory only once that block runs: each
    # kernel arrives at the cluster's barrier before its first load, and the join waits
    # for it before its first remote store
    join = (CSRC / "q4.cuh").read_text().split("void join(")[1]
    assert 0 <= join.find("cluster_wait();") < join.find("peer_store(part")
    for name in ("k_q4.cu", "k_q4_int.cu"):
        kernel = (CSRC / name).read_text().split("__global__")[1]
        assert 0 <= kernel.find("if (a.ks > 1) cluster_arrive();") < kernel.find("in.begin(a, at);"), name


@gpu
@pytest.mark.parametrize("xt,m,k,n,group", [("f32", 1, 20000, 40, 32), ("f32", 2, 70000, 20, 128), ("f32", 5, 9000, 64, 64),
                                            ("f16", 16, 16384, 256, 64), ("e4m3", 9, 30000, 30, 128)])
def test_q4_clusters_beside_other_work(cuda_mod, xt, m, k, n, group):
    # the blocks of a cluster start apart while other launches come and go
    a = Q4(xt, "f32", m, k, n, group, seed=31)
    a.call()
    a.check()
    want = a.y.clone()
    other, big = torch.cuda.Stream(), torch.zeros(1 << 22, device="cuda")
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(other):
            big.add_(1.0)
        a.y.zero_()
        a.call()
        assert torch.equal(a.y, want)
