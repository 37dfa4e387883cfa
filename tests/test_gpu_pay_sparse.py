"""pay_sparse_attention with the tensors that pay_attention takes: any layout of q, k and v gives the result of contiguous ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


def rnd(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(BF)


def odd_start(t):
    """the same values 2 bytes off a 16-byte border"""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


LAYOUTS = {"heads outside": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "channels outside": lambda t: t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0),
           "tokens outside": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "heads apart": lambda t: torch.cat([t, t], 3)[..., :128],
           "slice of a fused tensor": lambda t: torch.stack([t, t], 2)[:, :, 0], "odd rows": lambda t: torch.cat([t.flatten(2), t[:, :, 0, :4]], 2)[:, :, : t.shape[2] * 128].unflatten(2, (-1, 128)),
           "odd start": odd_start, "backwards and back": lambda t: t.flip(1).flip(1)}


@pytest.mark.parametrize("B,Lq,Lk,H,Hk", [(2, 300, 500, 4, 4), (2, 300, 500, 4, 2), (1, 1, 200, 3, 1), (3, 17, 64, 1, 1), (2, 1, 1, 2, 2)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_any_layout(ops, layout, B, Lq, Lk, H, Hk):
    q, k, v = rnd(1, B, Lq, H, 128), rnd(2, B, Lk, Hk, 128), rnd(3, B, Lk, Hk, 128)
    ref = ops.pay_sparse_attention([q, k, v], 3)
    of = LAYOUTS[layout]
    assert torch.equal(of(q), q)
    assert torch.equal(ops.pay_sparse_attention([of(q), of(k), of(v)], 3), ref)
    assert torch.equal(ops.pay_sparse_attention([of(q), k, of(v)], 3, recycle_q=True), ref)


def test_one_row_for_all(ops):
    """broadcast views: a token, a head, a batch that stands for all"""
    q, k, v = rnd(4, 2, 200, 4, 128), rnd(5, 2, 300, 4, 128), rnd(6, 2, 300, 4, 128)
    for view in (q[:, :1].expand(-1, 200, -1, -1), q[:, :, :1].expand(-1, -1, 4, -1), q[:1].expand(2, -1, -1, -1)):
        assert torch.equal(ops.pay_sparse_attention([view, k, v], 2), ops.pay_sparse_attention([view.contiguous(), k, v], 2))
    for view in (k[:, :1].expand(-1, 300, -1, -1), k[:, :, :1].expand(-1, -1, 4, -1), k[:1].expand(2, -1, -1, -1)):
        assert torch.equal(ops.pay_sparse_attention([q, view, v], 2), ops.pay_sparse_attention([q, view.contiguous(), v], 2))


@pytest.mark.parametrize("B,Lq,Lk", [(0, 200, 300), (2, 0, 300), (2, 200, 0), (0, 0, 0)])
def test_nothing_to_attend(ops, B, Lq, Lk):
    q, k, v = rnd(7, B, Lq, 2, 128), rnd(8, B, Lk, 2, 128), rnd(9, B, Lk, 2, 128)
    qm, km = ops.block_mean(q, 128), ops.block_mean(k, 64)
    index, count = ops.select_blocks(qm, km, 3)
    assert index.shape == (B, 2, (Lq + 127) // 128, 3) and count.shape == index.shape[:3]
    if Lk == 0:
        assert (index == -1).all() and (count == 0).all()
    o = ops.pay_sparse_attention([q, k, v], 3)
    assert o.shape == q.shape and o.dtype == BF and (o == 0).all()


@pytest.mark.parametrize("keep", [0, -1])
def test_no_blocks_to_keep_is_refused(ops, keep):
    from wan2gp_amd.lib import WanHipError
    q = rnd(10, 1, 200, 2, 128)
    with pytest.raises(WanHipError, match="keep"):
        ops.select_blocks(ops.block_mean(q, 128), ops.block_mean(q, 64), keep)
    with pytest.raises(WanHipError, match="keep"):
        ops.pay_sparse_attention([q, q, q], keep)
