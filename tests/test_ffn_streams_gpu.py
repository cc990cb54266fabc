"""Streams other than the one that owns a layer's memory, on the GPU."""
import pytest
import torch

from ffn_util import moe_ref
from gpu_util import note
from test_moe_gpu import _close, _layer, _make, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("current", [False, True])
def test_a_layer_dropped_while_a_stream_works_on_it(lk, current):
    """The workspace is the layer's own: dropped with the layer while a side stream has still to
    run, its memory is not handed to the next allocation."""
    hidden, ffn, E, k, T = 256, 128, 8, 2, 20
    L = _layer(95, E, hidden, ffn)
    layer = _make(lk, L, k, max_tokens=T)
    keep = layer._keep                                   # the weights are the caller's tensors
    x = _x(96, T, hidden, torch.float32).cuda()
    out = torch.empty_like(x)
    a = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    note(f"a layer dropped while a side stream works, current {current}")
    with torch.cuda.stream(side):
        for _ in range(20):                              # some 20 ms before the layer's turn
            torch.mm(a, a, out=b)
        if current:
            layer(x, out)
    if not current:
        layer(x, out, stream=side)
    at, n = layer._work.data_ptr(), layer._work.numel()
    del layer
    new = torch.empty(n, dtype=torch.uint8, device="cuda")
    early, other = not side.query(), new.data_ptr() != at
    torch.cuda.synchronize()
    assert early and other                               # nothing is written to it: the choices lie there
    _close(out, moe_ref(x.cpu(), k=k, score="sigmoid", **L)[0], torch.float32, "dropped layer")
    del keep


class _Elsewhere:
    """A stream of a device that the tensors are not on."""
    device_index, cuda_stream = 1, 0x1000


def test_a_stream_of_another_device_is_refused(lk):
    x = torch.ones(2, 64, device="cuda")
    q, sc = lk.i8_rows(2, 64), torch.ones(2, device="cuda")
    layer = _make(lk, _layer(97, 2, 64, 32), 1, max_tokens=2)
    note("a stream of another device")
    for call in (lambda: lk.norm_q8(x, torch.ones(64, device="cuda"), q, sc, stream=_Elsewhere()),
                 lambda: lk.gemm_i8(q, sc, q, sc, torch.empty(2, 2, device="cuda"), stream=_Elsewhere()),
                 lambda: layer(x, x, stream=_Elsewhere())):
        with pytest.raises(ValueError, match="another device"):
            call()


def test_captured_on_the_layers_own_workspace(lk):
    """A graph of calls on the layer's own workspace, replayed between eager calls on another
    stream in order; the layer goes after the graph."""
    hidden, ffn, E, k, T = 256, 128, 8, 2, 20
    layer = _make(lk, _layer(98, E, hidden, ffn), k, max_tokens=T)
    x, out = torch.empty(T, hidden, device="cuda"), torch.empty(T, hidden, device="cuda")
    x.copy_(_x(99, T, hidden, torch.float32))
    note("a layer captured on its own workspace")
    layer(x, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(x, out)
    for rep in range(4):
        x.copy_(_x(110 + rep, T, hidden, torch.float32))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        side, want = torch.cuda.Stream(), torch.empty_like(out)
        torch.cuda.synchronize()
        layer(x, want, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, want), rep
    del g, layer
    torch.cuda.synchronize()
    torch.empty(1 << 20, device="cuda").zero_()
    torch.cuda.synchronize()
