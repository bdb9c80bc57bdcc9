"""Waits that run out, in calls through the torch binding: nothing faults, and the caller is told."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

WAIT_CYCLES = 2_000_000      # about a millisecond of SM clock


def test_a_wait_that_ran_out_is_told_by_the_next_call(cuda):
    """A product whose copies from the third block of the contracted axis on are left out gives up. Whichever operator is
    called next says so, once; the library-wide word is not touched."""
    import rocal_b200
    from rocal_b200._lib import lib
    from rocal_b200._torch import head
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(5)
    x, w = (torch.randn((n, 512), generator=g, device=cuda).half() for n in (40, 200))
    labels, grad = torch.zeros(40, dtype=torch.int32, device=cuda), torch.ones(10, device=cuda)
    want = P.linear(x, w)

    def gives_up():
        head.linear_raw(x, w, None, None, "none", None, False, None, (WAIT_CYCLES, 2), watched=True)
        torch.cuda.synchronize()
    for call in (lambda: P.linear(x, w), lambda: P.linear_cross_entropy(x, w, labels), lambda: P.clip_grad_norm([grad], 0.5), P.check_unfinished):
        gives_up()
        with pytest.raises(rocal_b200.Rb200Error, match="unfinished"):
            call()
        call()
        assert bool((grad == grad[0]).all()) and torch.equal(P.linear(x, w), want)
        grad.fill_(1)
    # in a captured graph, too, whose replays raise the same word
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        head.linear_raw(x, w, None, None, "none", None, False, None, (WAIT_CYCLES, 2), watched=True)
    P.check_unfinished()
    for _ in range(2):
        graph.replay()
        with pytest.raises(rocal_b200.Rb200Error, match="unfinished"):
            P.check_unfinished()
    assert lib.rb200k_device_status() == 0



def test_the_longest_sums_are_waited_for(cuda):
    """A tile's products of 2^29 contracted elements (within the documented extents) take more than a second of SM clock, the
    limit of ordinary waits: 8.4 million blocks of 64 elements at 290 clocks or more. Values are zero but for a few, so that the
    sums are exact."""
    from rocal_b200 import kernels as K
    k = 1 << 29
    x, w = torch.zeros((1, k), dtype=torch.bfloat16, device=cuda), torch.zeros((2, k), dtype=torch.bfloat16, device=cuda)
    x[0, 0], x[0, k // 2 + 1], x[0, -1] = 3.0, 5.0, 7.0
    w[0, 0], w[0, k // 2 + 1], w[1, -1], w[1, 5] = 2.0, 1.0, 1.5, 9.0
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    loss, stats, info = K.linear_cross_entropy(x, w, torch.ones(1, dtype=torch.int64, device=cuda), reduction="sum", status=status)
    assert int(status) == 0 and float(stats[0]) == 11.0 and float(stats[2]) == 10.5                # scores 11 and 10.5
    assert abs(float(loss) - (11.0 - 10.5 + torch.log1p(torch.exp(torch.tensor(-0.5, dtype=torch.float64))).item())) <= 1e-6


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("n,k,v", [(100, 256, 90), (40000, 256, 90), (40000, 128, 128), (300, 512, 200), (2000, 640, 3000)])
def test_waits_of_the_loss_run_out(cuda, n, k, v, backward):
    """Copies from the second block of the features on are left out, in the way for few classes (tiles fewer and more than the SMs) and in the
    general one: every role gives up, the status word reads 1, and the next call on the same buffers is right."""
    import ctypes
    from rocal_b200 import kernels as K
    from rocal_b200._lib import LinearCeParams, lib
    g = torch.Generator(device=cuda).manual_seed(n + k + v)
    x, w = (torch.randn((r, k), generator=g, device=cuda).half() / 8 for r in (n, v))
    labels = torch.randint(0, v, (n,), generator=g, device=cuda)
    loss, stats, info = K.linear_cross_entropy(x, w, labels, reduction="sum")
    grads = K.linear_cross_entropy_backward(torch.ones_like(loss), x, w, labels, stats, info, reduction="sum")
    status, one = torch.zeros(1, dtype=torch.int32, device=cuda), torch.ones((), device=cuda)
    outs = [torch.zeros_like(t) for t in (loss, stats, info) + grads]
    p = LinearCeParams()
    p.dtype, p.reduction, p.rows, p.features, p.classes, p.label_bytes, p.ignore_index = 1, 2, n, k, v, 8, -100
    p.x, p.ldx, p.weight, p.ldw, p.labels = x.data_ptr(), k, w.data_ptr(), k, labels.data_ptr()
    p.loss, p.stats, p.info, p.dloss = outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), one.data_ptr()
    p.dx, p.lddx, p.dweight, p.lddw, p.dbias, p.status = outs[3].data_ptr(), k, outs[4].data_ptr(), k, outs[5].data_ptr(), status.data_ptr()
    need = (lib.rb200k_linear_ce_backward_workspace_bytes if backward else lib.rb200k_linear_ce_workspace_bytes)(ctypes.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    stream = torch.cuda.current_stream().cuda_stream
    if backward:
        outs[1].copy_(stats)
        outs[2].copy_(info)
    for skip, cycles, told in ((1, WAIT_CYCLES, 1), (0, WAIT_CYCLES, 1), (-1, WAIT_CYCLES * 1000, 0)):
        status.zero_()
        assert lib.rb200k_linear_ce_probe(ctypes.byref(p), stream, int(backward), cycles, skip) == 0
        torch.cuda.synchronize()
        assert int(status) == told, skip
    for got, want in zip(outs[3:], grads) if backward else zip(outs[:2], (loss, stats)):
        assert torch.equal(got, want)
