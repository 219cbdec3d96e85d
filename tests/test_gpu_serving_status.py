"""A bounded wait of the serving operators that runs out is told by
kk_serving_status, once, and by no other call."""
import numpy as np
import pytest

import kokopop_b200 as kb
from test_gpu_serving import KK, _stream

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _product(ctx, stream):
    w = torch.full((20, 64), 0x99, dtype=torch.uint8, device="cuda")  # every weight 1
    sc, x = torch.ones(20, 1, device="cuda").half(), torch.ones(1, 128, device="cuda")
    out = torch.empty(1, 20, device="cuda")
    torch.cuda.synchronize()
    ctx.q4_matvec_device(1, 20, 128, 128, w.data_ptr(), sc.data_ptr(), KK["f32"], x.data_ptr(), 128, 0,
                         out.data_ptr(), 20, stream)
    ctx.serving_status(stream)
    return out


def test_status_of_calls_that_finished_is_ok(ctx):
    for stream in (0, _stream(), torch.cuda.Stream().cuda_stream):
        assert bool((_product(ctx, stream) == 128).all())


def test_a_wait_that_runs_out_is_told_once_and_by_the_status_alone(ctx):
    """The tight wait of 2 ms on a barrier that nothing arrives at; the
    synthesis does not take the failure for its own."""
    from kokopop_b200 import workload as W
    ctx.upload(W.config2_weights())
    utts = [W.make_utterance(np.random.default_rng(9), 7)]
    want = ctx.decoder_forward(utts)
    side = torch.cuda.Stream()
    for stream in (0, side.cuda_stream):
        assert ctx.L.kk_serving_wait_selftest(ctx.h, 2000, stream) == kb.KK_OK  # asynchronous, like the operators
        torch.cuda.synchronize()
        np.testing.assert_array_equal(ctx.decoder_forward(utts)[0], want[0])
        with pytest.raises(kb.KKError) as e:
            ctx.serving_status(stream)
        assert e.value.code == kb.KK_ERROR_INFERENCE and "bounded wait ran out" in str(e.value)
        ctx.serving_status(stream)
        assert bool((_product(ctx, stream) == 128).all())


def test_a_synthesis_failure_is_not_told_by_the_status(ctx):
    assert ctx.L.kk_wait_selftest(ctx.h, 2000) == kb.KK_ERROR_INFERENCE
    ctx.serving_status(_stream())


def test_status_is_refused_while_the_stream_is_captured(ctx):
    graph, side, x = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(kb.KKError) as e:
            ctx.serving_status(torch.cuda.current_stream().cuda_stream)
        x += 1.0
    assert e.value.code == kb.KK_ERROR_INVALID_ARGUMENT
    graph.replay()
    ctx.serving_status(_stream())
    assert bool((x == 1.0).all())
