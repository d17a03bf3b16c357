"""Outputs that lie over inputs are refused where they are not named as places for them, and column ranges of one wider matrix beside each other are not
such.  The checks come before anything asks for a device: host memory stands in for the GPU's."""
import pytest
import torch

from aici_amd._lib import HipAttnError, call
from aici_amd.kernels import _desc


def desc(t):
    return _desc(t, device=False)


def linear(out, x, w, scale, bias=None, residual=None):
    call("hipattn_linear_fp8", desc(out), desc(x), desc(w), desc(scale), desc(bias), desc(residual), None, None)


def accepted(run):
    """Whether the arguments pass (without a device the call then ends where it asks for one)."""
    if torch.cuda.is_available():
        pytest.skip("host memory, which only a machine without a GPU may be handed")
    try:
        run()
    except HipAttnError as e:
        return "lies over" not in str(e) and "must" not in str(e)
    return True


@pytest.mark.parametrize("m", [1, 2, 20, 300])
def test_linear_fp8(m):
    n, k = 272, 256
    store = torch.zeros((1 << 20,), dtype=torch.bfloat16)
    x = torch.zeros((m, k), dtype=torch.bfloat16)
    out = store[:m * n].view(m, n)
    raw = store.view(torch.uint8)
    w, scale, bias = torch.zeros((n, k), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones((3, 2)), torch.zeros((n,), dtype=torch.bfloat16)
    with pytest.raises(HipAttnError, match="out lies over weight"):
        linear(out, x, raw[:n * k].view(torch.float8_e4m3fn).view(n, k), scale)
    with pytest.raises(HipAttnError, match="out lies over weight"):  # its last rows
        last = 2 * m * n - 16
        linear(out, x, raw[last:last + n * k].view(torch.float8_e4m3fn).view(n, k), scale)
    with pytest.raises(HipAttnError, match="out lies over weight_scale"):
        linear(out, x, w, raw[16:16 + 24].view(torch.float32).view(3, 2))
    with pytest.raises(HipAttnError, match="out lies over bias"):
        linear(out, x, w, scale, bias=out[0])
    for first in (4, (m - 1) * n + 4):  # some of it, or another row's
        with pytest.raises(HipAttnError, match="out lies over part of residual"):
            linear(out, x, w, scale, residual=store[first:first + m * n].view(m, n))
    if m > 1:
        with pytest.raises(HipAttnError, match="out lies over part of residual"):
            linear(out, x, w, scale, residual=out[:1].expand(m, n))
        with pytest.raises(HipAttnError, match="out lies over part of residual"):
            linear(out, x, w, scale, residual=store[:2 * m * n].view(m, 2 * n)[:, :n])
    assert accepted(lambda: linear(out, x, w, scale, bias=bias, residual=out))
    wide = store[:m * (2 * n + k)].view(m, 2 * n + k)
    assert accepted(lambda: linear(wide[:, :n], wide[:, 2 * n:], w, scale, bias=bias, residual=wide[:, n:2 * n]))
    assert accepted(lambda: linear(store[:m * n].view(m, n), store[:m * k].view(m, k), w, scale, bias=bias))


def tree(out, q, kc, vc, tables, cu, ctx, mask):
    call("hipattn_paged_attention_tree", desc(q), desc(kc), desc(vc), desc(tables), desc(cu), desc(ctx), 4, 40, 0.1, desc(mask), desc(out), None, None)


def test_paged_attention_tree():
    T, hq, hkv, d, bs, blocks = 8, 4, 2, 64, 16, 6
    store = torch.zeros((1 << 16,), dtype=torch.float16)
    out, elements = store[:T * hq * d].view(T, hq, d), T * hq * d
    good = {"q": torch.zeros((T, hq, d), dtype=torch.float16), "kc": torch.zeros((blocks, hkv, d // 8, bs, 8), dtype=torch.float16),
            "vc": torch.zeros((blocks, hkv, d, bs), dtype=torch.float16), "tables": torch.zeros((2, 3), dtype=torch.int32),
            "cu": torch.tensor([0, 4, 8], dtype=torch.int32), "ctx": torch.tensor([40, 9], dtype=torch.int32), "mask": torch.zeros((T, 1), dtype=torch.int64)}
    for name, operand in (("q", "q"), ("kc", "key_cache"), ("vc", "value_cache"), ("tables", "block_tables"), ("cu", "cu_seqlens_q"),
                          ("ctx", "context_lens"), ("mask", "tree_mask")):
        t = good[name]
        for first in (16, 2 * elements - 16):
            place = store.view(torch.uint8)[first:first + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
            with pytest.raises(HipAttnError, match=f"out lies over (part of )?{operand}"):
                tree(out, **{**good, name: place})
    with pytest.raises(HipAttnError, match="out lies over part of q"):  # its heads in another order
        tree(out, **{**good, "q": store[:elements].view(hq, T, d).transpose(0, 1)})
    assert accepted(lambda: tree(out, **good))
    assert accepted(lambda: tree(out, **{**good, "q": out}))
    wide = store[:2 * elements].view(T, 2, hq, d)
    assert accepted(lambda: tree(wide[:, 1], **{**good, "q": wide[:, 0]}))
    heads = store[:3 * elements].view(T, hq, 3, d)  # every head's q beside its k and v
    assert accepted(lambda: tree(heads[:, :, 2], **{**good, "q": heads[:, :, 0]}))
    assert accepted(lambda: tree(heads[:, :, 0], **{**good, "q": heads[:, :, 2]}))
    with pytest.raises(HipAttnError, match="out lies over part of q"):
        tree(store[32:32 + 3 * elements].view(T, hq, 3, d)[:, :, 0], **{**good, "q": heads[:, :, 0]})


def test_tree_accept():
    kc, vc = torch.zeros((4, 2, 8, 16, 8), dtype=torch.float16), torch.zeros((4, 2, 64, 16), dtype=torch.float16)
    i32 = [torch.zeros((4,), dtype=torch.int32) for _ in range(3)]
    cu, slots, ptrs = torch.tensor([0, 4], dtype=torch.int32), torch.zeros((4,), dtype=torch.int32), torch.zeros((2,), dtype=torch.int64)
    one, path = torch.zeros((1,), dtype=torch.int32), torch.zeros((1, 4), dtype=torch.int32)

    def accept(lens=one, path=path, following=torch.zeros((1,), dtype=torch.int32)):
        call("hipattn_tree_accept", *map(desc, i32), desc(cu), 4, desc(slots), desc(ptrs), desc(ptrs.clone()), desc(kc), desc(vc), desc(lens), desc(path),
             desc(following), None)

    for kw in ({"lens": ptrs.view(torch.int32)[1:2]}, {"path": ptrs.view(torch.int32).view(1, 4)}, {"following": ptrs.view(torch.int32)[3:]}):
        with pytest.raises(HipAttnError, match="an output lies over an input"):
            accept(**kw)
    assert accepted(accept)
