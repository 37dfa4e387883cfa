"""Block-sparse attention on the GPU against plain 64-bit forms: block_mean, select_blocks, sparse_attention and the three together.

Tolerances, from the roundings that the operators make (a rounding to bf16 is off by at most 2^-8 of the value, to fp32 2^-24):
  block_mean        summed in 64 bits, rounded once to fp32
  select_blocks     whole numbers: equal
  sparse_attention  q * scale is rounded to bf16, so a score is off by at most 2^-8 A, A = max_j sum_i |q_i k_ji| / sqrt(128), and a weight by a
                    factor e^(2^-8 A); the weights are rounded to bf16 in the product with v (2^-8) and not in their sum.  Numerator and
                    denominator: |o - o'| <= (2^-8 + 2 (e^(2^-8 A) - 1)) sum_j p_j |v_j| + (n + 200) 2^-24 sum_j p_j |v_j| for n keys in fp32 sums,
                    and 2^-8 |o| for the output's rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCALE = 1 / math.sqrt(128)


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rnd(g, *shape, gain=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * gain).to(BF)


def lens_of(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def mean_ref(x, block, lens=None):
    B, L, H, D = x.shape
    n = (L + block - 1) // block
    out = torch.zeros(B, H, n, D, dtype=F64, device=x.device)
    for b in range(B):
        end = L if lens is None else min(max(int(lens[b]), 0), L)
        for i in range(n):
            rows = x[b, i * block : max(i * block, min((i + 1) * block, end))].to(F64)
            if len(rows):
                out[b, :, i] = rows.mean(0)
    return out


def select_ref(qm, km, keep, lens=None):
    B, H, nq, _ = qm.shape
    Bk, Hk, nk, _ = km.shape
    index = torch.full((B, H, nq, keep), -1, dtype=torch.int32)
    count = torch.zeros(B, H, nq, dtype=torch.int32)
    qm, km = qm.cpu().to(F64), km.cpu().to(F64)
    for b in range(B):
        n = nk if lens is None else min(max((int(lens[b % Bk]) + 63) // 64, 0), nk)
        for h in range(H):
            s = (qm[b, h][:, None, :] * km[b % Bk, h // (H // Hk)][None, :n, :]).sum(2)
            for r in range(nq):
                # NaN above everything, equal scores: the lowest block first
                order = sorted(range(n), key=lambda j: (0 if math.isnan(s[r, j]) else 1, 0 if math.isnan(s[r, j]) else -float(s[r, j]), j))[:keep]
                index[b, h, r, : len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
                count[b, h, r] = len(order)
    return index.cuda(), count.cuda()


def attend_ref(q, k, vt, index, count=None, lens=None, scale=SCALE):
    """(o, bound) in 64 bits"""
    B, Lq, H, D = q.shape
    Bk, Lk, Hk, _ = k.shape
    o = torch.zeros(B, Lq, H, D, dtype=F64, device=q.device)
    bound = torch.zeros_like(o)
    lists = index.cpu()
    for b in range(B):
        end = Lk if lens is None else min(max(int(lens[b % Bk]), 0), Lk)
        for h in range(H):
            kh = k[b % Bk, :, h // (H // Hk)].to(F64)
            vh = vt[b % Bk, (h // (H // Hk)) * 128 : (h // (H // Hk) + 1) * 128, :Lk].to(F64).t()
            for n in range(lists.shape[2]):
                c = lists.shape[3] if count is None else min(max(int(count[b, h, n]), 0), lists.shape[3])
                keys = []
                for j in lists[b, h, n, :c].tolist():
                    if 0 <= j:
                        keys += range(min(64 * j, end), min(64 * j + 64, end))
                if not keys:
                    continue
                keys = torch.tensor(keys, device=q.device)
                qq = q[b, 128 * n : 128 * n + 128, h].to(F64)
                p = torch.softmax(qq @ kh[keys].t() * scale, 1)
                A = (qq.abs() @ kh[keys].abs().t() * scale).amax()
                o[b, 128 * n : 128 * n + 128, h] = p @ vh[keys]
                mag = p @ vh[keys].abs()
                bound[b, 128 * n : 128 * n + 128, h] = (2.0 ** -8 + 2 * math.expm1(min(2.0 ** -8 * float(A), 50.0)) + (len(keys) + 200) * 2.0 ** -24) * mag
    return o, bound + 2.0 ** -8 * o.abs()


def check(got, ref, bound):
    assert torch.isfinite(got.float()).all()
    d = (got.to(F64) - ref).abs()
    bad = d > bound + 1e-30
    assert not bad.any(), (d[bad].max().item(), (d / (bound + 1e-30)).max().item(), bad.sum().item())


# ---- block_mean ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,L,H,block,lens", [(1, 1, 1, 128, None), (1, 64, 1, 64, None), (2, 65, 3, 64, [65, 0]), (1, 1000, 5, 128, None), (2, 777, 12, 64, [777, 301]),
                                              (1, 33, 40, 7, None), (3, 200, 2, 128, [1000, -5, 64]), (1, 4099, 1, 64, [4097])])
def test_block_mean(ops, B, L, H, block, lens):
    g = gen(L)
    x = rnd(g, B, L, H, 128) + 2.0
    if lens is not None:                     # what lies past a length is never read into a mean
        for b in range(B):
            x[b, min(max(lens[b], 0), L):] = float("nan")
    got = ops.block_mean(x, block, lens_of(lens))
    ref = mean_ref(x, block, lens)
    assert got.shape == ref.shape and got.dtype == F32
    assert ((got.to(F64) - ref).abs() <= 2.0 ** -24 * ref.abs() * 1.0001).all()


def test_block_mean_of_a_slice_of_a_fused_projection(ops):
    x = rnd(gen(3), 2, 333, 3, 4, 128)
    for i in range(3):
        assert torch.equal(ops.block_mean(x[:, :, i], 64), ops.block_mean(x[:, :, i].contiguous(), 64))


# ---- select_blocks ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,Bk,H,Hk,nq,nk,keep,lens", [(1, 1, 1, 1, 1, 1, 1, None), (1, 1, 2, 1, 3, 17, 5, None), (2, 2, 4, 2, 9, 65, 16, [4100, 130]), (2, 1, 3, 3, 5, 64, 64, None),
                                                       (1, 1, 1, 1, 70, 300, 37, None), (1, 1, 2, 2, 2, 30, 50, [0]), (2, 2, 1, 1, 4, 200, 1, [12800, 1]), (1, 1, 1, 1, 2, 1500, 600, None),
                                                       (1, 1, 1, 1, 2, 5000, 700, [319999]), (1, 1, 2, 1, 3, 20000, 900, None), (1, 1, 1, 1, 70, 2049, 2048, None), (2, 1, 3, 1, 17, 256, 30, [16300]), (1, 1, 2, 2, 33, 257, 256, None),
                                                       (1, 1, 3, 3, 16, 640, 64, None), (2, 2, 2, 1, 31, 641, 70, [41000, 0]), (1, 1, 5, 1, 49, 1216, 148, [77800]), (1, 1, 2, 1, 20, 1217, 148, None),
                                                       (3, 3, 1, 1, 15, 1180, 7, [1, 449, 75520])])
def test_select_blocks(ops, B, Bk, H, Hk, nq, nk, keep, lens):
    g = gen(nk + keep)
    qm = torch.randn(B, H, nq, 128, generator=g, device="cuda")
    km = torch.randn(Bk, Hk, nk, 128, generator=g, device="cuda")
    index, count = ops.select_blocks(qm, km, keep, lens_of(lens))
    ri, rc = select_ref(qm, km, keep, lens)
    assert torch.equal(count, rc) and torch.equal(index, ri)


def test_select_blocks_ties_go_to_the_lowest_block(ops):
    g = gen(1)
    qm = torch.randn(1, 1, 3, 128, generator=g, device="cuda")
    km = torch.randn(1, 1, 4, 128, generator=g, device="cuda").repeat(1, 1, 50, 1)      # every score fifty times
    for keep in (1, 7, 60, 130):
        index, count = ops.select_blocks(qm, km, keep)
        ri, rc = select_ref(qm, km, keep)
        assert torch.equal(index, ri) and torch.equal(count, rc)
    zero = torch.zeros_like(km)
    index, _ = ops.select_blocks(qm, zero, 9)
    assert torch.equal(index, torch.arange(9, dtype=torch.int32, device="cuda").expand(1, 1, 3, 9))
    signed = zero.clone()
    signed[:, :, ::2] = -0.0                                                            # -0 equals 0
    index, _ = ops.select_blocks(qm.abs(), signed, 9)
    assert torch.equal(index, torch.arange(9, dtype=torch.int32, device="cuda").expand(1, 1, 3, 9))


def test_select_blocks_nan_and_infinite_scores(ops):
    g = gen(2)
    qm = torch.rand(1, 1, 2, 128, generator=g, device="cuda") + 0.1
    km = torch.randn(1, 1, 40, 128, generator=g, device="cuda")
    km[0, 0, 5] = float("inf")
    km[0, 0, 7] = -float("inf")
    km[0, 0, 9, 3] = float("nan")
    for keep in (1, 2, 3, 39, 40):
        index, count = ops.select_blocks(qm, km, keep)
        ri, rc = select_ref(qm, km, keep)
        assert torch.equal(index, ri) and torch.equal(count, rc)
    assert ops.select_blocks(qm, km, 1)[0].flatten().tolist() == [9, 9]


# ---- sparse_attention ------------------------------------------------------------------------------------------------------------------
def lists(g, B, H, nq, nk, keep):
    """random lists without repetition, unsorted"""
    r = torch.rand(B, H, nq, max(nk, keep), generator=g, device="cuda")
    r[..., nk:] = -1
    idx = r.argsort(dim=3, descending=True)[..., :keep].to(torch.int32)
    return torch.where(idx < nk, idx, -1).contiguous()


def vt_of(v, fill=0.0):
    B, L, H, _ = v.shape
    vt = torch.full((B, H * 128, (L + 63) // 64 * 64), fill, dtype=BF, device=v.device)
    vt[:, :, :L] = v.permute(0, 2, 3, 1).reshape(B, H * 128, L)
    return vt


SHAPES = [(1, 1, 1, 1, 1, 1, 1, None), (1, 1, 1, 1, 1, 64, 1, None), (1, 1, 2, 1, 1, 1000, 7, None), (1, 1, 1, 1, 127, 65, 2, None), (1, 1, 3, 3, 128, 63, 1, None),
          (1, 1, 2, 2, 129, 640, 4, None), (2, 2, 4, 2, 300, 777, 5, [777, 100]), (2, 1, 4, 4, 257, 1500, 9, None), (2, 2, 5, 1, 128, 900, 20, [0, 899]),
          (1, 1, 1, 1, 64, 9000, 100, None), (4, 2, 2, 2, 40, 200, 3, [1, 65]), (1, 1, 8, 8, 1000, 2049, 12, None), (1, 1, 40, 8, 1, 20000, 64, [19999]),
          (1, 1, 2, 1, 200, 4096, 64, None), (1, 1, 1, 1, 16, 30000, 300, [29000])]


@pytest.mark.parametrize("B,Bk,H,Hk,Lq,Lk,keep,lens", SHAPES)
@pytest.mark.parametrize("gain", [1.0, 4.0])
def test_sparse_attention(ops, B, Bk, H, Hk, Lq, Lk, keep, lens, gain):
    g = gen(Lq + Lk)
    q, k, v = rnd(g, B, Lq, H, 128, gain=gain), rnd(g, Bk, Lk, Hk, 128), rnd(g, Bk, Lk, Hk, 128)
    nq, nk = (Lq + 127) // 128, (Lk + 63) // 64
    index = lists(g, B, H, nq, nk, keep)
    vt = vt_of(v)
    got = ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens))
    check(got, *attend_ref(q, k, vt, index, None, lens))


def test_sparse_attention_with_every_block_is_attention(ops):
    g = gen(9)
    q, k, v = rnd(g, 2, 513, 3, 128), rnd(g, 2, 1300, 3, 128), rnd(g, 2, 1300, 3, 128)
    index = torch.arange(21, dtype=torch.int32, device="cuda").expand(2, 3, 5, 21).contiguous()
    vt = ops.transpose_v(v)
    got = ops.sparse_attention(q, k, vt, index)
    ref, bound = attend_ref(q, k, vt, index)
    check(got, ref, bound)
    check(ops.attention(q, k, vt), ref, bound)


def test_masked_places_may_hold_anything(ops):
    """Keys past a batch's length, with K and V of infinities and NaN there; lists that name such blocks, blocks past the cache, negative ones."""
    g = gen(11)
    lens = [70, 700, 0]
    q, k, v = rnd(g, 3, 200, 2, 128), rnd(g, 3, 1000, 2, 128), rnd(g, 3, 1000, 2, 128)
    for b in range(3):
        k[b, lens[b]:] = float("nan")
        v[b, lens[b]:] = float("inf")
        k[b, lens[b] + 1 :: 2] = -float("inf")
    vt = vt_of(v, fill=float("nan"))
    index = torch.tensor([-1, 15, 1, 0, 99, 1 << 30, -(1 << 31), 10, 3], dtype=torch.int32, device="cuda").expand(3, 2, 2, 9).contiguous()
    got = ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens))
    clean_k, clean_vt = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(vt, 0, 0, 0)
    check(got, *attend_ref(q, clean_k, clean_vt, index, None, lens))
    assert (got[2] == 0).all()


def test_counts_and_repeated_blocks(ops):
    g = gen(12)
    q, k, v = rnd(g, 1, 400, 2, 128), rnd(g, 1, 640, 2, 128), rnd(g, 1, 640, 2, 128)
    index = lists(g, 1, 2, 4, 10, 10)
    index[..., 3] = index[..., 1]                                            # a block listed twice counts twice
    count = torch.tensor([[[0, 1, 4, 10], [11, -3, 2, 5]]], dtype=torch.int32, device="cuda")
    vt = vt_of(v)
    got = ops.sparse_attention(q, k, vt, index, count)
    check(got, *attend_ref(q, k, vt, index, count))
    assert (got[0, :128, 0] == 0).all() and (got[0, 128:256, 1] == 0).all()


def test_maxima_that_rise_along_the_list(ops):
    """Every block's scores lie far above (or below) those of the blocks before it: the running reference has to follow by more than one exponent range."""
    g = gen(13)
    for sign in (1, -1):
        k = rnd(g, 1, 1280, 1, 128, gain=0.02)
        k[0, :, 0, 0] += (torch.arange(1280, device="cuda") // 64 * 30 * sign).to(BF)
        q = rnd(g, 1, 130, 1, 128, gain=0.1)
        q[0, :, 0, 0] = 8.0
        q[0, ::3, 0, 0] = -8.0
        v = rnd(g, 1, 1280, 1, 128)
        index = torch.arange(20, dtype=torch.int32, device="cuda").expand(1, 1, 2, 20).contiguous()
        vt = vt_of(v)
        qs = (q.float() * ops.attention_qscale()).to(BF)                     # (the scale's own rounding is left out: scores of 400 would turn it into any weight)
        got = ops.sparse_attention(qs, k, vt, index, q_prescaled=True)
        check(got, *attend_ref(qs, k, vt, index, scale=math.log(2.0)))


def test_prescaled_queries_strides_and_in_place(ops):
    g = gen(14)
    fused = rnd(g, 2, 500, 3, 4, 128)
    q, k, v = fused[:, :, 0], fused[:, :, 1], fused[:, :, 2].contiguous()
    index = lists(g, 2, 4, 4, 8, 5)
    vt = vt_of(v)
    a = ops.sparse_attention(q, k, vt, index)
    assert torch.equal(a, ops.sparse_attention(q.contiguous(), k.contiguous(), vt, index))
    qc = q.contiguous()
    assert ops.sparse_attention(qc, k, vt, index, out=qc) is qc and torch.equal(qc, a)
    qs = (q.float() * ops.attention_qscale()).to(BF)
    check(ops.sparse_attention(qs, k, vt, index, q_prescaled=True), *attend_ref(qs, k, vt, index, scale=math.log(2.0)))


def test_long_cache_past_32_bit_offsets(ops):
    """k and vt of 2^31 elements and more each: the listed blocks lie at both ends."""
    g = gen(15)
    Lk, H = 430000, 40
    k = torch.zeros(1, Lk, H, 128, dtype=BF, device="cuda")
    vt = torch.zeros(1, H * 128, (Lk + 63) // 64 * 64, dtype=BF, device="cuda")
    q = rnd(g, 1, 3, H, 128)
    nk = (Lk + 63) // 64
    index = torch.tensor([0, nk - 2, nk - 1], dtype=torch.int32, device="cuda").expand(1, H, 1, 3).contiguous()
    for j in (0, nk - 2, nk - 1):
        n = min(64, Lk - 64 * j)
        k[0, 64 * j : 64 * j + n] = rnd(g, n, H, 128)
        vt[0, :, 64 * j : 64 * j + n] = rnd(g, H * 128, n)
    got = ops.sparse_attention(q, k, vt, index)
    check(got, *attend_ref(q, k, vt, index))
    m = ops.block_mean(k, 64)
    for j in (0, nk - 1):
        ref = k[0, 64 * j : 64 * j + 64].to(F64).mean(0)
        assert ((m[0, :, j].to(F64) - ref).abs() <= 2.0 ** -24 * ref.abs() * 1.0001).all()


@pytest.mark.parametrize("B,Bk,H,Hk,Lq,Lk,keep,lens", [(1, 1, 40, 8, 1700, 3000, 9, [2999]), (2, 1, 20, 20, 1665, 640, 4, [577]), (1, 1, 30, 1, 2300, 5000, 70, None),
                                                       (1, 1, 32, 2, 2048, 1000, 12, None)])
def test_more_lists_than_run_at_a_time(ops, B, Bk, H, Hk, Lq, Lk, keep, lens):
    """Whole rounds of lists, and what is left behind them cut into shares (none, a few, many); in place and with counts too."""
    g = gen(Lq + keep)
    q, k, v = rnd(g, B, Lq, H, 128), rnd(g, Bk, Lk, Hk, 128), rnd(g, Bk, Lk, Hk, 128)
    nq = (Lq + 127) // 128
    index = lists(g, B, H, nq, (Lk + 63) // 64, keep)
    count = torch.randint(0, keep + 1, (B, H, nq), generator=g, device="cuda", dtype=torch.int32)
    vt = vt_of(v, fill=float("nan"))
    got = ops.sparse_attention(q, k, vt, index, count, k_lens=lens_of(lens))
    check(got, *attend_ref(q, k, vt_of(v), index, count, lens))
    assert ops.sparse_attention(q, k, vt, index, count, k_lens=lens_of(lens), out=q) is q and torch.equal(q, got)


def test_output_over_an_input_is_refused(ops):
    from wan2gp_amd.lib import WanHipError
    g = gen(41)
    for L in (12, 200):
        both = rnd(g, 2, 1, L, 2, 128)
        q, k, v = both[0], both[1], rnd(g, 1, L, 2, 128)
        vt, index = vt_of(v), torch.zeros(1, 2, (L + 127) // 128, 1, dtype=torch.int32, device="cuda")
        ref = ops.sparse_attention(q, k, vt, index)
        for out in (k, both.view(-1)[256 : 256 + q.numel()].view_as(q), vt.view(-1)[: q.numel()].view_as(q)):
            with pytest.raises(WanHipError, match="overlap"):
                ops.sparse_attention(q, k, vt, index, out=out)
        fused = rnd(g, 1, L, 2, 2, 128)                                          # a strided q, and an output over its memory
        with pytest.raises(WanHipError, match="overlap"):
            ops.sparse_attention(fused[:, :, 0], k, vt, index, out=fused.view(-1)[: q.numel()].view_as(q))
        assert ops.sparse_attention(q, k, vt, index, out=q) is q and torch.equal(q, ref)


# ---- up to 16 queries: a kernel of their own ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,Bk,H,Hk,Lq,Lk,keep,lens", [(1, 1, 1, 1, 1, 1, 1, None), (2, 1, 6, 2, 2, 65, 3, None), (2, 2, 5, 1, 15, 2000, 31, [2000, 63]), (1, 1, 40, 8, 16, 9000, 141, [8999]),
                                                       (1, 1, 40, 8, 17, 9000, 141, [8999]), (3, 3, 400, 4, 1, 640, 9, [1, 64, 640]), (1, 1, 1, 1, 1, 75600, 1182, None),
                                                       (1, 1, 4, 2, 7, 16000, 250, None), (1, 1, 1, 1, 5, 256, 4, None), (1, 1, 1, 1, 5, 320, 5, None)])
def test_few_queries(ops, B, Bk, H, Hk, Lq, Lk, keep, lens):
    """Both sides of the limit; one workgroup to a list and many, one block a wave and several; in place, strided, with counts."""
    g = gen(Lq * 7 + keep)
    fused = rnd(g, B, Lq, H, 2, 128)
    q, k, v = fused[:, :, :, 0].contiguous(), rnd(g, Bk, Lk, Hk + 1, 128)[:, :, :Hk], rnd(g, Bk, Lk, Hk, 128)
    index = lists(g, B, H, 1, (Lk + 63) // 64, keep)
    count = torch.randint(0, keep + 2, (B, H, 1), generator=g, device="cuda", dtype=torch.int32)
    vt = vt_of(v, fill=float("nan"))
    clean = vt_of(v)
    check(ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens)), *attend_ref(q, k, clean, index, None, lens))
    got = ops.sparse_attention(q, k, vt, index, count, k_lens=lens_of(lens))
    check(got, *attend_ref(q, k, clean, index, count, lens))
    assert (got.permute(0, 2, 1, 3)[count[:, :, 0] == 0] == 0).all()
    assert ops.sparse_attention(q, k, vt, index, count, k_lens=lens_of(lens), out=q) is q and torch.equal(q, got)


@pytest.mark.parametrize("Lq", [1, 16])
def test_few_queries_masked_places_may_hold_anything(ops, Lq):
    g = gen(21)
    lens = [70, 700, 0]
    q, k, v = rnd(g, 3, Lq, 2, 128), rnd(g, 3, 1000, 2, 128), rnd(g, 3, 1000, 2, 128)
    for b in range(3):
        k[b, lens[b]:] = float("nan")
        v[b, lens[b]:] = float("inf")
        k[b, lens[b] + 1 :: 2] = -float("inf")
    vt = vt_of(v, fill=float("nan"))
    index = torch.tensor([-1, 15, 1, 0, 99, 1 << 30, -(1 << 31), 10, 3], dtype=torch.int32, device="cuda").expand(3, 2, 1, 9).contiguous()
    got = ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens))
    check(got, *attend_ref(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(vt, 0, 0, 0), index, None, lens))
    assert (got[2] == 0).all()


def test_few_queries_keep_a_nan_that_is_attended(ops):
    g = gen(22)
    q, k, v = rnd(g, 1, 3, 1, 128), rnd(g, 1, 640, 1, 128), rnd(g, 1, 640, 1, 128)
    k[0, 70, 0, 5] = float("nan")
    vt = vt_of(v)
    for entries in ([1], [1, 0], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9]):
        index = torch.tensor(entries, dtype=torch.int32, device="cuda").view(1, 1, 1, -1)
        assert torch.isnan(ops.sparse_attention(q, k, vt, index)).all()
    index = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda").view(1, 1, 1, -1)
    check(ops.sparse_attention(q, k, vt, index), *attend_ref(q, torch.nan_to_num(k), vt, index))


def test_few_queries_maxima_that_rise_along_the_list(ops):
    g = gen(23)
    for sign in (1, -1):
        k = rnd(g, 1, 19200, 1, 128, gain=0.02)
        k[0, :, 0, 0] += (torch.arange(19200, device="cuda") // 64 * 2 * sign).to(BF)
        q = rnd(g, 1, 9, 1, 128, gain=0.1)
        q[0, :, 0, 0] = 8.0
        q[0, ::3, 0, 0] = -8.0
        v = rnd(g, 1, 19200, 1, 128)
        index = torch.arange(300, dtype=torch.int32, device="cuda").view(1, 1, 1, 300)
        vt = vt_of(v)
        qs = (q.float() * ops.attention_qscale()).to(BF)
        check(ops.sparse_attention(qs, k, vt, index, q_prescaled=True), *attend_ref(qs, k, vt, index, scale=math.log(2.0)))


def test_few_queries_captured_beside_another_graph(ops):
    g = gen(24)
    state = []
    for n in range(2):
        q, k, v = rnd(g, 1, 1, 8, 128), rnd(g, 1, 4000, 2, 128), rnd(g, 1, 4000, 2, 128)
        vt, index = vt_of(v), lists(g, 1, 8, 1, 63, 40)
        ops.sparse_attention(q, k, vt, index)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sparse_attention(q, k, vt, index)
        state.append((graph, q, k, vt, index, out))
    for turn in range(3):
        for graph, q, *_ in state:
            q.copy_(rnd(g, 1, 1, 8, 128))
        for graph, *_ in state:
            graph.replay()
        torch.cuda.synchronize()
        for graph, q, k, vt, index, out in state:
            assert torch.equal(out, ops.sparse_attention(q, k, vt, index))


def test_long_cache_past_32_bit_offsets_of_many_queries(ops):
    g = gen(25)
    Lk, H = 430000, 40
    k = torch.zeros(1, Lk, H, 128, dtype=BF, device="cuda")
    vt = torch.zeros(1, H * 128, (Lk + 63) // 64 * 64, dtype=BF, device="cuda")
    q = rnd(g, 1, 130, H, 128)
    nk = (Lk + 63) // 64
    index = torch.tensor([0, nk - 2, nk - 1], dtype=torch.int32, device="cuda").expand(1, H, 2, 3).contiguous()
    for j in (0, nk - 2, nk - 1):
        n = min(64, Lk - 64 * j)
        k[0, 64 * j : 64 * j + n] = rnd(g, n, H, 128)
        vt[0, :, 64 * j : 64 * j + n] = rnd(g, H * 128, n)
    check(ops.sparse_attention(q, k, vt, index), *attend_ref(q, k, vt, index))


# ---- together ---------------------------------------------------------------------------------------------------------------------------
def test_pay_sparse_attention(ops):
    g = gen(16)
    q, k, v = rnd(g, 2, 700, 4, 128), rnd(g, 2, 700, 4, 128), rnd(g, 2, 700, 4, 128)
    lens = [700, 130]
    qkv = [q.clone(), k, v]
    got = ops.pay_sparse_attention(qkv, 3, k_lens=lens_of(lens))
    assert qkv == [] and got.dtype == BF
    qm, km = ops.block_mean(q, 128), ops.block_mean(k, 64, lens_of(lens))
    index, count = select_ref(qm, km, 3, lens)
    check(got, *attend_ref(q, k, vt_of(v), index, count, lens))
    assert ops.pay_sparse_attention([q.float(), k.float(), v.float()], 3).dtype == F32
    one = ops.pay_sparse_attention([q, k[:1], v[:1]], 3)                         # k / v batch 1 is broadcast
    two = ops.pay_sparse_attention([q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1)], 3)
    assert torch.equal(one, two)
    assert (ops.pay_sparse_attention([q, k[:, :0], v[:, :0]], 3) == 0).all()
    same = ops.pay_sparse_attention([q, q.clone(), v], 3)                        # one tensor as q and k: its storage is not reused
    keep = q.clone()
    assert torch.equal(ops.pay_sparse_attention([q, q, v], 3, recycle_q=True), same) and torch.equal(q, keep)
    got = ops.pay_sparse_attention([q, k, v], 3, recycle_q=True)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, ops.pay_sparse_attention([keep, k, v], 3))


def test_captured_and_replayed_beside_another_graph(ops):
    """Two graphs of the same calls, replayed in turn on new inputs with eager work between: every replay equals the eager result."""
    g = gen(17)
    lens = lens_of([1900])
    state = []
    for n in range(2):
        q, k, v = rnd(g, 1, 200, 3, 128), rnd(g, 1, 2000, 3, 128), rnd(g, 1, 2000, 3, 128)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.pay_sparse_attention([q, k, v], 6, k_lens=lens)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.pay_sparse_attention([q, k, v], 6, k_lens=lens)
        state.append((graph, q, k, v, out))
    for turn in range(3):
        for graph, q, k, v, out in state:
            q.copy_(rnd(g, 1, 200, 3, 128)); k.copy_(rnd(g, 1, 2000, 3, 128)); v.copy_(rnd(g, 1, 2000, 3, 128))
            lens.fill_(1900 - 700 * turn)
        for graph, *_ in state:
            graph.replay()
        torch.cuda.synchronize()
        for graph, q, k, v, out in state:
            assert torch.equal(out, ops.pay_sparse_attention([q, k, v], 6, k_lens=lens))


def test_on_another_stream(ops):
    g = gen(18)
    q, k, v = rnd(g, 1, 900, 2, 128), rnd(g, 1, 3000, 2, 128), rnd(g, 1, 3000, 2, 128)
    ref = ops.pay_sparse_attention([q, k, v], 9)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([ops.pay_sparse_attention([q, k, v], 9) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for per in outs for o in per)
