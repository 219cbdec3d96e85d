"""Serving calls return to the host at once, whatever is queued on the GPU."""
import time

import numpy as np
import pytest

from test_gpu_serving import _stream
from test_gpu_token_stream import _attend, _decode_setup

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_divided_attention_does_not_wait_on_the_host_for_synthesis_before_it(ctx):
    """A synthesis call queued behind half a second of other work leaves its
    uploads in flight; the attention calls after it use no upload and return
    before that work is done. They run after the synthesis (one workspace)."""
    from kokopop_b200 import workload as W
    ctx.upload(W.config2_weights())
    n, asr, f0, noise, style = W.pack([W.make_utterance(np.random.default_rng(9), 7)])
    dev = [torch.from_numpy(a).cuda() for a in (asr, f0, noise, style)]
    audio = torch.empty(600 * int(n.sum()), device="cuda")
    s = _decode_setup(2, 6000, 16, 8, 2, 64)
    want, out = torch.zeros_like(s[1]), torch.zeros_like(s[1])
    side = torch.cuda.Stream()

    def synthesis(stream):
        ctx.decoder_forward_device(n, *(d.data_ptr() for d in dev), audio.data_ptr(), stream)

    synthesis(side.cuda_stream)  # warm: nothing is allocated below
    _attend(ctx, s, want, _stream())
    torch.cuda.synchronize()
    first = audio.clone()
    length = int(s[3].max())
    view, q, table, lens, cu, _ = s
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(0.5 * 1.9e9))
    t0 = time.perf_counter()
    synthesis(side.cuda_stream)
    for _ in range(3):
        ctx.paged_attention_device(view, q.shape[0], lens.data_ptr(), cu.data_ptr(), q.shape[0], 1, length,
                                   table.data_ptr(), table.shape[1], q.data_ptr(), q.stride(0), q.shape[1], 0.125, 0,
                                   out.data_ptr(), out.stride(0), _stream())
    t1 = time.perf_counter()
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    assert t2 - t0 > 0.3, "the work before was too short to tell"
    assert t1 - t0 < 0.5 * (t2 - t0)
    assert torch.equal(out, want) and torch.equal(audio, first)
