"""Several host threads on one stream, and on hipStreamPerThread: tree attention and linear layers of 8-bit weights hand partial results and rounded
rows from one launch to the next in the library's scratch memory, and still get their own.  Every output has the bits of a call alone."""
import ctypes
import threading

import pytest
import torch

from aici_amd import kernels as K
from aici_amd._lib import call
from aici_amd.kernels import _desc

from test_gpu_trees import Case

pytestmark = pytest.mark.gpu
CALLS, THREADS = 100, 2
PER_THREAD_STREAM = 2  # hipStreamPerThread


def operator(name, seed, device):
    """(the output's shape, call(out, stream))."""
    if name == "tree":
        c = Case(seed, [24, 7, 40], [1500, 900, 2000], (32, 8, 128), 16, torch.bfloat16, device)
        q, kc, vc, tables, cu, ctx, most, max_k, scale, mask = args = c.args()
        made = [_desc(t) for t in (q, kc, vc, tables, cu, ctx, mask)]

        def run(out, stream, args=args):
            call("hipattn_paged_attention_tree", *made[:6], most, max_k, scale, made[6], _desc(out), None, stream)
        return tuple(q.shape), run
    rows = int(name.split()[1])
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, 4096), generator=g).to(torch.bfloat16).to(device)
    w, scale = (t.to(device) for t in K.quantize_weight_fp8(torch.randn((1024, 4096), generator=g)))
    made = [_desc(t) for t in (x, w, scale)]

    def run(out, stream, keep=(x, w, scale)):
        call("hipattn_linear_fp8", _desc(out), *made, None, None, None, stream)
    return (rows, 1024), run


@pytest.mark.parametrize("stream", ["one stream", "a stream of each thread's own"])
@pytest.mark.parametrize("name", ["tree", "linear 9", "linear 100", "linear 300"])
def test_threads(device, name, stream):
    made = [operator(name, seed, device) for seed in (3, 4)]
    side = torch.cuda.Stream()
    handle = ctypes.c_void_p(side.cuda_stream if stream == "one stream" else PER_THREAD_STREAM)
    outs = [torch.zeros((CALLS, *shape), dtype=torch.bfloat16, device=device) for shape, _ in made]
    alone = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for shape, _ in made]
    first = torch.cuda.Stream()  # (its own scratch memory, as the one stream's)
    torch.cuda.synchronize()
    for (_, run), out in zip(made, alone):
        run(out, handle if stream == "one stream" or name != "tree" else ctypes.c_void_p(first.cuda_stream))
        torch.cuda.synchronize()
    errors = []

    def calls(k):
        try:
            for out in outs[k]:
                made[k][1](out, handle)
            torch.cuda.ExternalStream(handle.value).synchronize()  # (a thread's own stream goes with it, and nobody else waits for what it still does)
        except Exception as e:  # (shown by the test, not lost with its thread)
            errors.append(e)

    threads = [threading.Thread(target=calls, args=(k,)) for k in range(THREADS)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for out, want in zip(outs, alone):
        if name == "tree" and stream != "one stream":
            # There contexts are whole: other last bits, the same for every call.  Each is off by u (A + |out|) and little more, u = 2^-8 and both
            # at most 1 where a row sees 900 keys and more: 4 u and a quarter.
            assert float((out[0].double() - want.double()).abs().max()) <= 5 * 2.0 ** -8
            want = out[0]
        assert bool((out == want).all())
