"""Both sides of each size at which another kernel of the choice of blocks takes over, and every kernel of the block-sparse attention and of the MXFP4 Linears captured into
graphs that are replayed in turn."""
import pytest
import torch

from test_gpu_sparse_attention import BF, F64, gen, lists, rnd, vt_of
from test_gpu_sparse_attention import ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nk", [255, 256, 257, 511, 512, 513, 767, 768, 769, 1023, 1024, 1025, 1279, 1280, 1281, 1535, 1536, 1537, 1791, 1792, 1793, 2047, 2048, 2049, 6799, 6800, 6801])
def test_select_blocks_at_the_kernels_borders(ops, nk):
    """Whole numbers below 2^24 as means: every score is exact and many are equal, so which of them are taken is the lists' whole content."""
    g = gen(nk)
    B, H, nq, keep = 2, 2, 21, nk // 5 + 3
    qm = torch.randint(-3, 4, (B, H, nq, 128), generator=g, device="cuda").float()
    km = torch.randint(-3, 4, (B, H, nk, 128), generator=g, device="cuda").float()
    lens = [nk * 64 - 5, (nk // 2) * 64 + 1]
    index, count = ops.select_blocks(qm, km, keep, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    score = qm.double() @ km.double().transpose(2, 3).contiguous()
    for b in range(B):
        n = (lens[b] + 63) // 64
        best = torch.sort(score[b, ..., :n], dim=2, descending=True, stable=True)[1][..., :keep].sort(2)[0]
        c = min(keep, n)
        assert (count[b] == c).all() and torch.equal(index[b, ..., :c].long(), best) and (index[b, ..., c:] == -1).all()


def attention_call(ops, g, Lq, Lk, H, Hk, keep):
    q, k, v = rnd(g, 1, Lq, H, 128), rnd(g, 1, Lk, Hk, 128), rnd(g, 1, Lk, Hk, 128)
    vt, index = vt_of(v), lists(g, 1, H, (Lq + 127) // 128, (Lk + 63) // 64, keep)
    return q, lambda: ops.sparse_attention(q, k, vt, index)


def linear_call(ops, g, M, N, K, epilogue):
    x, w, b = rnd(g, M, K), rnd(g, N, K, gain=K ** -0.5), rnd(g, N)
    wm = ops.mxfp4_quantize(w)
    more = dict(residual=rnd(g, M, N), mod=rnd(g, 6, N), e=rnd(g, 1, 6, N), gate_idx=1) if epilogue == 2 else {}
    return x, lambda: ops.linear_mxfp4(x, *wm, b, epilogue=epilogue, **more)


def pay_call(ops, g, L, keep):
    q, k, v = rnd(g, 1, L, 2, 128), rnd(g, 1, L, 2, 128), rnd(g, 1, L, 2, 128)
    return q, lambda: ops.pay_sparse_attention([q, k, v], keep)


CALLS = {"few queries in shares": lambda o, g: attention_call(o, g, 3, 9000, 8, 2, 100), "few queries": lambda o, g: attention_call(o, g, 16, 200, 4, 4, 3),
         "lists in shares": lambda o, g: attention_call(o, g, 200, 6000, 2, 2, 90), "whole lists": lambda o, g: attention_call(o, g, 2048, 700, 32, 32, 3),
         "whole lists and shares": lambda o, g: attention_call(o, g, 2300, 3000, 30, 30, 40), "choice in one launch": lambda o, g: pay_call(o, g, 3000, 5), "choice in two": lambda o, g: pay_call(o, g, 17000, 9),
         "few rows": lambda o, g: linear_call(o, g, 5, 1024, 1024, 0), "parts along K": lambda o, g: linear_call(o, g, 40, 256, 5120, 1), "small tiles": lambda o, g: linear_call(o, g, 600, 1536, 768, 2),
         "large tiles": lambda o, g: linear_call(o, g, 9001, 1160, 1056, 2), "large tiles, transposed": lambda o, g: linear_call(o, g, 9000, 1160, 256, 3)}


@pytest.mark.parametrize("name", CALLS)
def test_captured_and_replayed(ops, name):
    """Two graphs of a call, replayed in turn on inputs that change, with eager calls and synchronisations between: every replay is the eager result, bit for bit."""
    g = gen(len(name))
    graphs = []
    for _ in range(2):
        x, call = CALLS[name](ops, g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, x, call, out))
    for turn in range(4):
        for _, x, _, _ in graphs:
            x.copy_(rnd(g, *x.shape))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, x, call, out in graphs:
            assert torch.equal(out, call()), turn
