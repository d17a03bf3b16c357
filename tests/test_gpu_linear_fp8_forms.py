"""Every form that linear_fp8's product can take, at ragged sizes: the tolerance of test_gpu_linear_fp8.py, whose shapes leave some of them out.  `form`
restates the choice of linear_fp8.hip (plan_fp8), so that the list here can be seen to be whole."""
import pytest
import torch

from aici_amd import kernels as K

from test_gpu_linear_fp8 import check, operands

gpu = pytest.mark.gpu


def form(m, n, k):
    """("held" or "few", wavefronts to a tile of 16 rows of the weight), or the number of the tile."""
    kb = (k + 127) // 128
    if m <= 16:
        per, tiles = 1, (n + 15) // 16
        while per < 8 and kb // (2 * per) >= 2 and (tiles * per < 768 or (kb > 16 * per and tiles * per <= 1024)):
            per *= 2
        return "held" if m <= 2 and m * ((2 * k + 1023) // 1024 * 1024) <= 32 * 1024 else "few", per
    if m <= 32:
        return 0 if n < 4800 else 1 if n < 16384 else 2
    if m <= 64:
        return 3 if n < 4800 else 4 if n <= 8192 else 5 if n < 16384 else 6
    if m <= 128:
        return 7 if n < 16384 else 8
    large, small = -(-m // 256) * -(-n // 256), -(-m // 128) * -(-n // 128)
    us, tile = -(-large // 256) * 2.25 * kb, 10
    for s in range(1, 9):
        if s > 1 and kb // s < 4:
            break
        t = -(-small * s // 512) * -(-kb // s) * (1.2 if small * s <= 256 else 1.37) + (4 + m * n * s * (8 / 3.5e6) if s > 1 else 0)
        if t < us:
            us, tile = t, 9
    return tile


SHAPES = [  # weights that end inside a tile, columns that end inside a block; few and many stages of the ring
    (1, 16400, 272), (2, 6160, 400), (2, 6160, 4112), (1, 4096, 4112), (1, 272, 4112), (1, 4096, 14336), (2, 144, 2064),
    (5, 16400, 272), (16, 8208, 400), (4, 6160, 4112), (16, 4112, 4112), (9, 272, 4112), (16, 144, 14336),
    (20, 272, 400), (31, 4112, 4112), (20, 6160, 400), (24, 6160, 4112), (31, 16400, 272), (17, 16400, 4112),
    (50, 272, 656), (64, 4112, 4112), (33, 4816, 400), (48, 8176, 4112), (37, 10256, 400), (60, 8208, 4112), (50, 16400, 656), (63, 16400, 4112),
    (65, 272, 400), (127, 6160, 4112), (100, 16400, 272), (70, 16400, 4112),
    (129, 272, 400), (301, 4112, 4112), (4097, 272, 400), (2050, 6160, 656),
]


def test_every_form_is_there():
    found = {form(*s) for s in SHAPES}
    assert found == {(kind, per) for kind in ("held", "few") for per in (1, 2, 4, 8)} | set(range(11)), found


@gpu
@pytest.mark.parametrize("loud", [False, True], ids=["plain", "loud"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forms(device, m, n, k, dtype, loud):
    x, w, scale, g = operands(m + n + k, m, n, k, dtype, device, loud)
    out = K.linear_fp8(x, w, scale)
    check(out, x, w, scale, loud=loud)
    assert torch.equal(out, K.linear_fp8(x, w, scale))


@gpu
@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if s[2] in (400, 656, 272, 2064)])
def test_epilogues_and_places(device, m, n, k):
    """Bias and residual, out over the residual, over x, and beside x in rows of one wider matrix; what lies around out stays."""
    x, w, scale, g = operands(7, m, n, k, torch.bfloat16, device, loud=False)
    bias, residual = (torch.randn(s, generator=g).bfloat16().to(device) for s in ((n,), (m, n)))
    y = K.linear_fp8(x, w, scale, bias=bias, residual=residual)
    check(y, x, w, scale, bias, residual, loud=False)
    into = residual.clone()
    assert torch.equal(K.linear_fp8(x, w, scale, bias=bias, residual=into, out=into), y)
    wide = torch.full((m + 1, k + n + 16), 5.0, dtype=x.dtype, device=device)  # (rows of out on 8-byte boundaries, no wider ones)
    wide[:m, 8 + n:8 + n + k] = x
    beside = K.linear_fp8(wide[:m, 8 + n:8 + n + k], w, scale, bias=bias, residual=residual, out=wide[:m, 4:4 + n])
    assert torch.equal(beside, y) and torch.equal(wide[:m, 8 + n:8 + n + k], x)
    assert all(bool((part == 5).all()) for part in (wide[m:], wide[:, :4], wide[:, 4 + n:8 + n], wide[:, 8 + n + k:]))
    over = torch.zeros((m * max(n, k),), dtype=x.dtype, device=device)
    over[:m * k] = x.flatten()
    assert torch.equal(K.linear_fp8(over[:m * k].view(m, k), w, scale, bias=bias, residual=residual, out=over[:m * n].view(m, n)), y)


@gpu
@pytest.mark.parametrize("m", [1, 2])
def test_out_beside_x(device, m):
    """One or two rows: their columns and those of out in rows of one wider matrix share nothing, and x needs no rounded copy."""
    n, k = 272, 512
    x, w, scale, _ = operands(5, m, n, k, torch.float16, device)
    want = K.linear_fp8(x, w, scale)
    check(want, x, w, scale)
    wide = torch.zeros((m, k + n), dtype=x.dtype, device=device)
    wide[:, :k] = x
    assert torch.equal(K.linear_fp8(wide[:, :k], w, scale, out=wide[:, k:]), want) and torch.equal(wide[:, :k], x)


@gpu
@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if s[2] in (400, 656, 272)])
def test_rows_with_nan_and_infinity(device, m, n, k):
    """Such a row is NaN, the others are what they are without it."""
    x, w, scale, _ = operands(13, m, n, k, torch.bfloat16, device)
    want = K.linear_fp8(x, w, scale)
    odd = {0: float("nan"), m // 2: float("inf"), m - 1: -float("inf")}
    for row, v in odd.items():
        x[row, (37 * row + 5) % k] = v
    out = K.linear_fp8(x, w, scale)
    rest = [row for row in range(m) if row not in odd]
    assert bool(torch.isnan(out[list(odd)]).all()) and torch.equal(out[rest], want[rest])
