"""Several host threads on one stream, and on hipStreamPerThread: calls that hand partial results from one launch to the next in the library's
scratch memory still get their own.  Each thread calls with inputs of its own, over and over; every output has the bits of a call alone."""
import ctypes
import threading

import pytest
import torch

from aici_amd import kernels as K
from aici_amd import workloads as W
from aici_amd._lib import call
from aici_amd.kernels import _desc

pytestmark = pytest.mark.gpu
CALLS, THREADS = 150, 2
PER_THREAD_STREAM = 2  # hipStreamPerThread


def operator(name, seed, device):
    """(shape and type of the output, call(out, stream))."""
    g = torch.Generator().manual_seed(seed)
    if "decode" in name:
        d = W.decode_inputs(seed, 3, 1500, 2000, 8, 2, 128, torch.bfloat16, 400).to(device)
        tensors = [_desc(t) for t in (d.q, d.key_cache, d.value_cache, d.block_tables, d.context_lens)]

        def run(out, stream, d=d):
            q, kc, vc, tables, lens = tensors
            if name.startswith("window"):
                call("hipattn_paged_attention_window", _desc(out), q, kc, vc, 2, d.scale, tables, lens, 16, d.max_ctx, 1200, 20, None, None, stream)
            else:
                call("hipattn_paged_attention_v1", _desc(out), q, kc, vc, 2, d.scale, tables, lens, 16, d.max_ctx, None, stream)
        return (tuple(d.q.shape), torch.bfloat16), run
    if name == "linear":
        x, w = (torch.randn(s, generator=g).to(torch.bfloat16).to(device) for s in ((40, 4096), (1024, 4096)))
        assert K.linear_workspace_size(x, w) > 0
        keep = [x, w, _desc(x), _desc(w)]
        return ((40, 1024), torch.bfloat16), lambda out, stream: call("hipattn_linear", _desc(out), *keep[2:], None, None, None, stream)
    logits = torch.randn((5, 32768), generator=g).to(torch.bfloat16).to(device)
    mask = torch.randint(0, 256, (5, 4096), generator=g, dtype=torch.uint8).to(device)
    keep = [logits, mask, _desc(logits), _desc(mask)]
    return ((5,), torch.int32), lambda out, stream: call("hipattn_bias_argmax", keep[2], None, keep[3], None, _desc(out), None, stream)


@pytest.mark.parametrize("stream", ["one stream", "a stream of each thread's own"])
@pytest.mark.parametrize("name", ["window decode", "window decode, flat", "decode", "decode, flat", "linear", "argmax"])
def test_threads(device, tuning, name, stream):
    tuning("decode_flat", 1 if "flat" in name else 0)
    made = [operator(name, seed, device) for seed in range(THREADS)]
    if stream == "one stream":
        side = torch.cuda.Stream()
        handle = ctypes.c_void_p(side.cuda_stream)
    else:
        handle = ctypes.c_void_p(PER_THREAD_STREAM)
    alone, outs = [], []
    for (shape, dtype), run in made:
        outs.append(torch.zeros((CALLS, *shape), dtype=dtype, device=device))
        alone.append(torch.zeros(shape, dtype=dtype, device=device))
    torch.cuda.synchronize()
    for (_, run), out in zip(made, alone):
        run(out, handle)
        torch.cuda.synchronize()
    errors = []

    def calls(k):
        try:
            for out in outs[k]:
                made[k][1](out, handle)
        except Exception as e:  # (shown by the test, not lost with its thread)
            errors.append(e)

    threads = [threading.Thread(target=calls, args=(k,)) for k in range(THREADS)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert not torch.equal(alone[0], alone[1]) and bool(alone[0].any())
    for k in range(THREADS):
        assert all(torch.equal(out, alone[k]) for out in outs[k])
