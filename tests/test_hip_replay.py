"""Gradient buffers that kernels accumulate into are cleared inside the captured step: a graph is replayed several times, with eager
work between the replays, and each replay equals the eager call."""
import glob
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from conftest import REPO                                                  # noqa: E402


def test_no_memset_in_code_that_a_graph_may_record():
    """A memset node has left old sums in place on later replays; kernels clear instead."""
    for path in glob.glob(os.path.join(REPO, "subspace-reg_amd", "csrc", "*.hip")):
        with open(path) as f:
            assert not re.search(r"\bhipMemset\w*\s*\(", f.read()), path


@pytest.mark.gpu
@pytest.mark.parametrize("ksize,dtype", [(1, "bf16"), (3, "f32"), (1, "f32")])
def test_replayed_conv_wgrad_starts_from_zero(ksize, dtype):
    """The dW kernels that add with atomics.  With images of +-1 each sum is an integer below
    2^24, so any order of the additions is exact."""
    from subreg_hip import _lib
    lib = _lib.load()
    B, H, W, Cin, Cout = 4, 12, 12, 32, 64
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    code = _lib.BF16 if dtype == "bf16" else _lib.F32
    rng = np.random.RandomState(3)
    x = torch.from_numpy(rng.choice([-1.0, 1.0], (B * H * W, Cin))).to(td).cuda()
    dy = torch.from_numpy(rng.choice([-1.0, 1.0], (B * H * W, Cout))).to(td).cuda()
    splits = lib.subreg_conv_wgrad_splits(B, H, W, Cin, Cout, ksize, code)
    gw = torch.empty(splits * Cout * ksize * ksize * Cin, dtype=torch.float32, device="cuda")

    def run():
        _lib.check(lib.subreg_conv_wgrad(_lib.ptr(x), _lib.ptr(dy), _lib.ptr(gw), None, None, B, H, W, Cin, Cout, ksize, code,
                                         _lib.stream_ptr()))
    gw.fill_(float("nan"))
    run()
    torch.cuda.synchronize()
    want = gw.clone()
    if ksize == 1:
        grad = torch.empty(Cout, Cin, 1, 1, device="cuda")
        _lib.check(lib.subreg_unpack_wgrad(_lib.ptr(gw), _lib.ptr(grad), Cout, Cin, 1, 0, splits, _lib.stream_ptr()))
        assert torch.equal(grad.double().cpu().view(Cout, Cin), dy.double().cpu().t() @ x.double().cpu())
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        run()
    for i in range(6):
        gw.fill_(float(i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gw, want), i
        run()                                                              # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(gw, want), i
