"""The block bookkeeping of a step on the device (kernels.step_blocks) against lists, step after step: equal numbers everywhere, no block in
two places, what does not fit refused in the same words."""
import numpy as np
import pytest
import torch

from aici_amd import kernels as K
from aici_amd import paged
from oracle import steps

pytestmark = pytest.mark.gpu


def compare(got, want, dev_tables, model):
    for name, value in want.items():
        assert getattr(got, name).tolist() == value, name
    assert dev_tables.tolist() == model.tables


def random_lens(rng, R, hi, model):
    new = []
    for r in range(R):
        u = rng.random()
        new.append(-int(rng.integers(1, 5)) if u < 0.08 and model.kv[r] else 0 if u < 0.2 else 1 if u < 0.5 else int(rng.integers(1, hi + 1)))
    return new


@pytest.mark.parametrize("R,rows,per,hi,cols,nb,window,sinks,bs", [
    (1, 1, 0, 1, 3, 3, -1, 0, 16), (1, 40, 0, 70, 9, 9, 20, 3, 16), (7, 100, 0, 30, 12, 40, -1, 0, 8), (64, 64, 1, 1, 20, 300, 100, 4, 16),
    (65, 700, 10, 12, 20, 900, 33, 40, 16), (300, 3000, 0, 24, 12, 2500, 64, 0, 16), (300, 9000, 0, 90, 30, 4000, 100, 17, 32),
    (1024, 4096, 4, 4, 6, 3000, 50, 16, 16), (1500, 20000, 0, 40, 10, 9000, 90, 8, 16), (4096, 5000, 0, 3, 4, 9000, 10, 1, 8)])
def test_steps(device, R, rows, per, hi, cols, nb, window, sinks, bs):
    rng = np.random.default_rng(R + rows)
    model = steps.StepBlocks(bs, nb, R, cols, window, sinks)
    state = torch.zeros((R, 2), dtype=torch.int32, device=device)
    wide = torch.full((R, cols + 3), -9, dtype=torch.int32, device=device)
    tables = wide[:, :cols]
    tables.zero_()
    ring = torch.arange(nb, dtype=torch.int32, device=device)
    ends = torch.tensor([0, nb], dtype=torch.int64, device=device)
    for k in range(30 if R <= 100 else 8):
        new = random_lens(rng, R, hi, model)
        in_place = k % 2 == 1
        got = K.step_blocks(torch.tensor(new, dtype=torch.int32, device=device), state, tables, ring, ends, bs, rows, per, window, sinks,
                            *((state, ends) if in_place else ()))
        want = model.step(new, rows, per)
        compare(got, want, tables, model)
        assert ring.tolist() == model.ring
        state, ends = got.state, got.ends
        held = [model.tables[r][c] for r in range(R) for c in model.live(r)]
        assert len(held) + len(model.free) == nb and sorted(held + model.free) == list(range(nb))
    assert bool((wide[:, cols:] == -9).all())


def test_blocks_that_come_back_are_taken_in_the_same_step(device):
    """The pool is empty but for what ended requests and windows give back."""
    bs, R, cols, nb = 16, 40, 50, 600
    for rows in (4000, 30000):  # both launches
        model = steps.StepBlocks(bs, nb, R, cols, 64, 16)
        state = torch.zeros((R, 2), dtype=torch.int32, device=device)
        tables = torch.zeros((R, cols), dtype=torch.int32, device=device)
        ring = torch.arange(nb, dtype=torch.int32, device=device)
        ends = torch.tensor([0, nb], dtype=torch.int64, device=device)
        for new in ([480 if r < 20 else 0 for r in range(R)], [-1 if r < 3 else 0 if r < 20 else 32 for r in range(R)],
                    [500 if r < 4 else 40 for r in range(R)], [-1] * R):
            got = K.step_blocks(torch.tensor(new, dtype=torch.int32, device=device), state, tables, ring, ends, bs, max(rows, sum(x for x in new if x > 0)),
                                0, 64, 16)
            compare(got, model.step(new, max(rows, sum(x for x in new if x > 0))), tables, model)
            state, ends = got.state, got.ends
        assert got.totals.tolist() == [0, 0, nb, 0]


def test_replayed_steps(device):
    """A generation step captured once, its lengths kept on the device."""
    pool = paged.DeviceBlocks(16, 200, 12, 400, device, window_size_left=40, sink_tokens=4)
    model = steps.StepBlocks(16, 200, 12, 25, 40, 4)
    new = torch.zeros((12,), dtype=torch.int32, device=device)
    pool.step(new, 12, 1)
    model.step([0] * 12, 12, 1)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step = pool.step(new, 12, 1)
    rng = np.random.default_rng(1)
    for k in range(150):
        lens = [-1 if rng.random() < 0.02 else int(rng.random() < 0.9) for _ in range(12)]
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        want = model.step(lens, 12, 1)
        if k % 7 == 0:
            compare(step, want, pool.block_tables, model)
            assert pool.state.tolist() == want["state"] and pool.ring_ends.tolist() == want["ends"]
            torch.ones(1000, device=device).sum().item()


def test_states_that_are_none_stay_inside(device):
    """Nonsense in the state and the ring's ends gives nonsense, but no access outside the arrays, which lie in a frame."""
    R, cols, nb = 6, 5, 20
    frame = torch.full((3 * R * cols,), -5, dtype=torch.int32, device=device)
    tables = frame[R * cols:2 * R * cols].view(R, cols)
    rings = torch.full((3 * nb,), -6, dtype=torch.int32, device=device)
    state = torch.tensor([[2 ** 31 - 1, 2 ** 31 - 1], [-7, -7], [90, 2 ** 31 - 1], [79, -2 ** 31], [-2 ** 31, 3], [40, 1]], dtype=torch.int32,
                         device=device)
    for ends in ([0, 2 ** 40], [-5, 15], [2 ** 62, -2 ** 62], [30, 10]):
        for new in ([1, 1, 1, 1, 1, 1], [-1] * 6, [2 ** 31 - 1] * 6, [10, -1, 0, 1, 30, 30]):
            K.step_blocks(torch.tensor(new, dtype=torch.int32, device=device), state, tables, rings[nb:2 * nb],
                          torch.tensor(ends, dtype=torch.int64, device=device), 16, 64, 0, 3, 17)
    assert bool((frame[:R * cols] == -5).all()) and bool((frame[2 * R * cols:] == -5).all())
    assert bool((rings[:nb] == -6).all()) and bool((rings[2 * nb:] == -6).all())
