"""Cases of the operators that make a denoise step cheaper: self-attention over selected blocks of keys, and Linears in
microscaled 4-bit floating point.

`run` computes them in their plain form (elementary torch operations), or, with `own` set, through `wan2gp_amd.ops`:

  select    block_mean of q and k, then select_blocks: for each block of 128 queries the `keep` blocks of 64 keys whose mean key has
            the largest product with the block's mean query.
  attend    sparse_attention: softmax(q k^T / sqrt(128)) v over the listed blocks of keys.
  quantise  mxfp4_quantize, and mxfp4_dequantize back to the values that the codes stand for.
  linear    linear_mxfp4: x is quantised and multiplied with a weight that was quantised when it was loaded.
"""
import math

import torch

own = False

D = 128                     # head dimension of every attention here
QB, KB = 128, 64            # queries and keys of one block
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCALE = 1.0 / math.sqrt(D)


# ---- cases ---------------------------------------------------------------------------------------------------------------------
def listed():
    """480p x 81 frames is 21 x 30 x 52 = 32,760 tokens, 720p x 81 frames 21 x 45 x 80 = 75,600; one latent frame at 480p is 1,560.
    12 heads, 1,536 / 8,960 wide: the 1.3B model; 40 heads, 5,120 / 13,824 wide: the 14B model; 4,096 wide: its text tokens."""
    return [
        # one frame generated against the keys of the frames before it, two streams of which one is shorter
        dict(name="select-frame", op="select", B=2, H=12, Hk=12, Lq=1560, Lk=32760, keep=48, len0=32760, len1=17003),
        # a whole denoise step's choice of blocks at the largest resolution
        dict(name="select-720p", op="select", B=1, H=40, Hk=40, Lq=75600, Lk=75600, keep=148, len0=75600, len1=0),
        # one token against a long cache, five query heads to a key head: nothing but latency and the cache's bytes
        dict(name="attend-token", op="attend", B=1, H=40, Hk=8, Lq=1, Lk=75600, keep=32, len0=75600, len1=0),
        # the frame above
        dict(name="attend-frame", op="attend", B=2, H=12, Hk=12, Lq=1560, Lk=32760, keep=48, len0=32760, len1=17003),
        # the small model's self-attention at an eighth of the blocks
        dict(name="attend-480p", op="attend", B=1, H=12, Hk=12, Lq=32760, Lk=32760, keep=64, len0=32760, len1=0),
        # the large model's, likewise
        dict(name="attend-720p", op="attend", B=1, H=40, Hk=40, Lq=75600, Lk=75600, keep=148, len0=75600, len1=0),
        # the text tokens in front of the text embedding
        dict(name="quantise-text", op="quantise", M=512, K=4096),
        # the residual stream in front of the q / k / v Linears
        dict(name="quantise-720p", op="quantise", M=75600, K=5120),
        # the time projection: one row, all of it the weight's bytes
        dict(name="linear-time", op="linear", M=1, N=30720, K=5120, epilogue="none"),
        # the text embedding's first Linear with its GELU
        dict(name="linear-text", op="linear", M=512, N=5120, K=4096, epilogue="gelu"),
        # the small model's ffn.0
        dict(name="linear-480p", op="linear", M=32760, N=8960, K=1536, epilogue="gelu"),
        # the large model's ffn.2 with its gated residual
        dict(name="linear-720p", op="linear", M=75600, N=5120, K=13824, epilogue="gate"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("select", "attend", "attend", "quantise", "linear", "linear"))
    if op in ("select", "attend"):
        Hk = rng.choice((1, 2, 3, 4, 8, 12, 20))
        H = Hk * rng.choice((1, 1, 1, 2, 5)) if Hk < 12 else Hk
        B = rng.choice((1, 1, 2))
        Lk = _size(rng, 1, 75600)
        Lq = Lk if rng.random() < 0.5 else _size(rng, 1, 16384)
        keep = min(_size(rng, 1, 140 // B), (Lk + KB - 1) // KB + 2)
        lens = [Lk if rng.random() < 0.5 else rng.randint(0, Lk) for _ in range(B)]
        fused = Lq == Lk and H == Hk and rng.random() < 0.5                  # q and k side by side in one tensor
        return dict(op=op, B=B, H=H, Hk=Hk, Lq=Lq, Lk=Lk, keep=keep, len0=lens[0], len1=lens[1] if B > 1 else 0, fused=fused)
    if op == "quantise":
        return dict(op=op, M=_size(rng, 1, 60000), K=32 * _size(rng, 1, 200))
    K = 32 * _size(rng, 2, 432)
    return dict(op=op, M=_size(rng, 1, 40000), N=8 * _size(rng, 8, 1000), K=K, epilogue=rng.choice(("none", "gelu", "gate", "transposed")))


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(g, B, L, H, freq, phase):
    """What a normed, rotated projection looks like: noise on waves along the sequence, which the keys and queries of a head share."""
    x = torch.randn(B, L, H, D, generator=g, device="cuda", dtype=F32)
    for b in range(B):                                     # (a batch at a time: the angles of all of them need not be held at once)
        t = torch.arange(L, device="cuda", dtype=F32).view(L, 1, 1)
        x[b].mul_(0.8).add_(torch.cos(t * freq + phase), alpha=0.7)
    return x.to(BF16)


def _attention_inputs(case, g):
    B, H, Hk, Lq, Lk = case["B"], case["H"], case["Hk"], case["Lq"], case["Lk"]
    freq = torch.exp(-9.0 * torch.rand(1, Hk, D, generator=g, device="cuda")) * 0.6
    phase = 6.28 * torch.rand(1, Hk, D, generator=g, device="cuda")
    shared = H // Hk
    q = _tokens(g, B, Lq, H, freq.repeat_interleave(shared, 1), phase.repeat_interleave(shared, 1))
    k = _tokens(g, B, Lk, Hk, freq, phase)
    if case.get("fused"):
        qk = torch.stack([q, k], dim=2)
        q, k = qk[:, :, 0], qk[:, :, 1]
    ldv = (Lk + KB - 1) // KB * KB
    vt = torch.zeros(B, Hk * D, ldv, device="cuda", dtype=BF16)
    vt[:, :, :Lk] = torch.randn(B, Hk * D, Lk, generator=g, device="cuda", dtype=F32).to(BF16)
    lens = torch.tensor([case["len0"], case["len1"]][:B], dtype=torch.int32, device="cuda")
    return q, k, vt, lens


def _weight(g, N, K):
    """A weight quantised at load: codes [N, K / 2] and scales in the kernels' order."""
    w = torch.randn(N, K, generator=g, device="cuda", dtype=F32) * (1.0 / math.sqrt(K))
    codes, exps = _encode(w.to(BF16))
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8).contiguous(), _tile(exps)


def prepare(case, seed):
    g = _rng(seed)
    op = case["op"]
    if op in ("select", "attend"):
        q, k, vt, lens = _attention_inputs(case, g)
        state = dict(op=op, q=q, k=k, vt=vt, lens=lens, keep=case["keep"])
        if op == "attend":
            state["index"], state["count"] = _select(_block_mean(q, QB, None), _block_mean(k, KB, lens), case["keep"], lens)
        return state
    M, K = case["M"], case["K"]
    x = torch.randn(M, K, generator=g, device="cuda", dtype=F32) * torch.exp(1.5 * torch.randn(K, generator=g, device="cuda"))
    state = dict(op=op, x=x.to(BF16))
    del x
    if op == "linear":
        N = case["N"]
        state["epilogue"] = case["epilogue"]
        state["codes"], state["scales"] = _weight(g, N, K)
        state["bias"] = torch.randn(N, generator=g, device="cuda").to(BF16)
        if case["epilogue"] == "gate":
            state["residual"] = torch.randn(M, N, generator=g, device="cuda", dtype=F32).to(BF16)
            state["mod"] = torch.randn(6, N, generator=g, device="cuda").to(BF16)
            state["e"] = torch.randn(1, 6, N, generator=g, device="cuda").to(BF16)
    return state


# ---- 4-bit floating point in plain torch ---------------------------------------------------------------------------------------
# A block of 32 values along K shares the scale 2^e; a value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign.  e = exponent of the
# block's largest magnitude - 2, one more where that magnitude is 1.75 of its power of two or over (7 and over would be cut to 6).
def _encode(x):
    M, K = x.shape
    v = x.to(F32).view(M, K // 32, 32)
    bits = v.abs().amax(dim=2).view(torch.int32)
    e = (((bits + 0x200000) >> 23) - 129).clamp(-127, 125)
    y = torch.ldexp(v, -e.unsqueeze(2))
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code + 8 * torch.signbit(y)).view(M, K), (e + 127).to(torch.uint8)


def _decode(codes, exps):
    """codes [M, K] one to a byte, exps [M, K / 32] -> fp32 [M, K]"""
    M, K = codes.shape
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    return torch.ldexp(grid[codes.long()].view(M, K // 32, 32), exps.to(torch.int32).unsqueeze(2) - 127).view(M, K)


# Scales lie in tiles of 128 rows x 8 blocks (256 values of K), 1,024 bytes each, row tiles outside: inside a tile the byte of row r,
# block j is at [j & 3][r >> 3][j >> 2][r & 7].  Rows and blocks past the matrix are zeros.
def _tile(exps):
    M, J = exps.shape
    P, S = (M + 127) // 128, (J + 7) // 8
    full = torch.zeros(P * 128, S * 8, dtype=torch.uint8, device=exps.device)
    full[:M, :J] = exps
    return full.view(P, 16, 8, S, 2, 4).permute(0, 3, 5, 1, 4, 2).contiguous().view(-1)


def _untile(scales, M, K):
    P, S = (M + 127) // 128, (K // 32 + 7) // 8
    return scales.view(P, S, 4, 16, 2, 8).permute(0, 3, 5, 1, 4, 2).reshape(P * 128, S * 8)[:M, : K // 32]


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=2).view(packed.shape[0], -1)


# ---- the plain forms -----------------------------------------------------------------------------------------------------------
def _block_mean(x, block, lens):
    """[B, L, H, 128] -> fp32 [B, H, blocks, 128]: the mean of each block's rows below the batch's length, summed in 64 bits; 0 where there is none."""
    B, L, H, _ = x.shape
    n = (L + block - 1) // block
    end = torch.full((B, 1), L, device=x.device) if lens is None else lens.view(B, 1).long()
    seen = torch.arange(L, device=x.device) < end                                       # [B, L]
    full = torch.zeros(B, n * block, H, D, dtype=F64, device=x.device)
    full[:, :L] = torch.where(seen.view(B, L, 1, 1), x, 0).to(F64)
    rows = (end - torch.arange(n, device=x.device) * block).clamp(0, block)              # [B, n]
    return (full.view(B, n, block, H, D).sum(2) / rows.clamp(min=1).view(B, n, 1, 1)).to(F32).permute(0, 2, 1, 3).contiguous()


def _select(qm, km, keep, lens):
    """The `keep` best blocks of keys of each block of queries, ascending, -1 behind the last, and how many there are.  The scores are
    taken in 64 bits: in 32, which of two nearly equal ones wins would hang on the order of the sum."""
    B, H, nq, _ = qm.shape
    Hk, nk = km.shape[1], km.shape[2]
    k64 = km.to(F64).repeat_interleave(H // Hk, 1)
    score = torch.matmul(qm.to(F64), k64.transpose(2, 3).contiguous())                  # [B, H, nq, nk]
    valid = (lens.long() + KB - 1) // KB
    score = torch.where(torch.arange(nk, device=qm.device) < valid.view(B, 1, 1, 1), score, -math.inf)
    best = torch.sort(score, dim=3, descending=True, stable=True)[1][..., :keep]
    count = valid.clamp(max=keep).view(B, 1, 1).expand(B, H, nq)
    best = torch.where(torch.arange(best.shape[3], device=qm.device) < count.unsqueeze(3), best, nk)
    best = torch.sort(best, dim=3)[0]
    index = torch.full((B, H, nq, keep), -1, dtype=torch.int32, device=qm.device)
    index[..., : best.shape[3]] = torch.where(best < nk, best, -1)
    return index, count.to(torch.int32).contiguous()


def _attend(q, k, vt, index, lens):
    B, Lq, H, _ = q.shape
    Lk, Hk, ldv = k.shape[1], k.shape[2], vt.shape[2]
    nq, nk, keep = index.shape[2], ldv // KB, index.shape[3]
    qs = torch.zeros(B, H, nq * QB, D, dtype=F32, device=q.device)
    qs[:, :, :Lq] = q.permute(0, 2, 1, 3)
    ks = torch.zeros(B, Hk, nk * KB, D, dtype=BF16, device=q.device)
    ks[:, :, :Lk] = k.permute(0, 2, 1, 3)
    head = torch.arange(B * H, device=q.device)
    kv = head // H * Hk + head % H // (H // Hk)                                          # the row of k and v that a (batch, head) reads
    head, kv = head.repeat_interleave(nq), kv.repeat_interleave(nq)
    qs, ks = qs.view(B * H * nq, QB, D), ks.view(B * Hk, nk, KB, D)
    vs = vt.view(B * Hk, D, nk, KB).permute(0, 2, 3, 1)                                  # [B Hk, nk, 64, 128]
    idx = index.view(B * H * nq, keep).long()
    out = torch.empty(B * H * nq, QB, D, dtype=BF16, device=q.device)
    step = max(1, (1 << 32) // (keep * KB * D * 4))                                      # 4 GiB of gathered keys at a time
    for r in range(0, B * H * nq, step):
        i = idx[r : r + step]
        src, at = kv[r : r + step].unsqueeze(1), i.clamp(min=0)
        kg = ks[src, at].to(F32).reshape(-1, keep * KB, D)
        pos = (at.unsqueeze(2) * KB + torch.arange(KB, device=q.device))
        seen = (pos < lens.long()[head[r : r + step] // H].view(-1, 1, 1)) & (i >= 0).unsqueeze(2)
        vg = torch.where(seen.unsqueeze(3), vs[src, at], 0).to(F32).reshape(-1, keep * KB, D)
        s = torch.matmul(qs[r : r + step], kg.transpose(1, 2).contiguous()) * SCALE
        s = torch.where(seen.view(-1, 1, keep * KB), s, -math.inf)
        top = s.amax(dim=2, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(top), top, 0))
        total = p.sum(2, keepdim=True)
        out[r : r + step] = (torch.matmul(p, vg) / torch.where(total > 0, total, 1)).to(BF16)
    return out.view(B, H, nq * QB, D)[:, :, :Lq].permute(0, 2, 1, 3).contiguous()


def _linear(s):
    x, N = s["x"], s["codes"].shape[0]
    K = x.shape[1]
    w = _decode(_unpack(s["codes"]), _untile(s["scales"], N, K))
    y = torch.matmul(_decode(*_encode(x)), w.t()) + s["bias"].to(F32)
    if s["epilogue"] == "gelu":
        return (0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))).to(BF16)
    if s["epilogue"] == "gate":
        return (s["residual"].to(F32) + y * (s["mod"][GATE].to(F32) + s["e"][0, GATE].to(F32))).to(BF16)
    if s["epilogue"] == "transposed":
        M = x.shape[0]
        out = torch.zeros(N, (M + 63) // 64 * 64, dtype=BF16, device=x.device)
        out[:, :M] = y.t().to(BF16)
        return out
    return y.to(BF16)


GATE = 5                    # the row of the modulation that gates ffn.2


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "select":
        qm, km = _block_mean(s["q"], QB, None), _block_mean(s["k"], KB, s["lens"])
        return [qm, km, *_select(qm, km, s["keep"], s["lens"])]
    if s["op"] == "attend":
        return _attend(s["q"], s["k"], s["vt"], s["index"], s["lens"])
    if s["op"] == "quantise":
        return _decode(*_encode(s["x"])).to(BF16)
    return _linear(s)


def _run_own(s):
    from wan2gp_amd import lib, ops
    if s["op"] == "select":
        qm, km = ops.block_mean(s["q"], QB), ops.block_mean(s["k"], KB, s["lens"])
        return [qm, km, *ops.select_blocks(qm, km, s["keep"], k_lens=s["lens"])]
    if s["op"] == "attend":
        return ops.sparse_attention(s["q"], s["k"], s["vt"], s["index"], s["count"], k_lens=s["lens"])
    if s["op"] == "quantise":
        return ops.mxfp4_dequantize(*ops.mxfp4_quantize(s["x"]))
    if s["epilogue"] == "gate":
        return ops.linear_mxfp4(s["x"], s["codes"], s["scales"], s["bias"], lib.EPI_GATE_RES, residual=s["residual"], mod=s["mod"], e=s["e"], gate_idx=GATE)
    return ops.linear_mxfp4(s["x"], s["codes"], s["scales"], s["bias"], {"none": lib.EPI_NONE, "gelu": lib.EPI_GELU_TANH, "transposed": lib.EPI_TRANSPOSED}[s["epilogue"]])


def work(case):
    if case["op"] in ("select", "attend"):
        B, H, Hk, Lq, Lk, keep = (case[n] for n in ("B", "H", "Hk", "Lq", "Lk", "keep"))
        lens = [case["len0"], case["len1"]][:B]
        nq, nk = (Lq + QB - 1) // QB, (Lk + KB - 1) // KB
        if case["op"] == "select":
            n = B * Lq * H * D * 2 + sum(lens) * Hk * D * 2 + B * H * nq * D * 4 + B * Hk * nk * D * 4 + B * H * nq * (keep + 1) * 4
            return dict(bytes=n, flops=sum(2 * H * nq * ((n + KB - 1) // KB) * D for n in lens))
        seen = [min(keep * KB, n) for n in lens]                                # keys that a query attends
        touched = [min(n, H // Hk * nq * s) for n, s in zip(lens, seen)]        # keys of a head that any of its queries attends
        n = 2 * B * Lq * H * D * 2 + sum(2 * t * Hk * D * 2 for t in touched) + B * H * nq * keep * 4
        return dict(bytes=n, flops=sum(4 * H * Lq * s * D for s in seen))
    M, K = case["M"], case["K"]
    if case["op"] == "quantise":
        return dict(bytes=4 * M * K, flops=0)
    N = case["N"]
    n = 2 * M * K + N * K // 2 + N * K // 32 + 2 * N + 2 * M * N * (2 if case["epilogue"] == "gate" else 1)
    return dict(bytes=n, flops=2 * M * N * K)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def _round4(x):
    """bf16 -> the nearest values of its blocks' grids, in 64 bits: in [1, 8) of the scale a step is a half of the value's power of two."""
    M, K = x.shape
    v = x.to(F64).view(M, K // 32, 32)
    top = v.abs().amax(2, keepdim=True)
    m, p = torch.frexp(top)                                                     # top = m 2^p, m in [.5, 1)
    e = torch.where(top > 0, (p - 3 + (m >= 0.875)).clamp(-127, 125), -127).to(F64)
    y = v / 2.0 ** e
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return ((torch.round(y / step) * step).clamp(-6, 6) * 2.0 ** e).view(M, K)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "select":
        def mean(x, block, lens):
            B, L, H, _ = x.shape
            ends = [L] * B if lens is None else lens.tolist()
            parts = [[x[b, i : max(i, min(i + block, ends[b]))].to(F64) for i in range(0, L, block)] for b in range(B)]
            return torch.stack([torch.stack([p.mean(0) if len(p) else torch.zeros(H, D, dtype=F64, device="cuda") for p in row], 1) for row in parts])
        qm, km = mean(s["q"], QB, None), mean(s["k"], KB, s["lens"])
        return [qm, km, None, None]                                             # (which blocks are best: whole numbers, from the means in 32 bits)
    if s["op"] == "attend":
        q, k, vt = s["q"], s["k"], s["vt"]
        B, Lq, H, _ = q.shape
        shared, lists, ends = H // k.shape[2], s["index"].cpu(), s["lens"].tolist()
        out = torch.zeros(B, Lq, H, D, dtype=F64, device="cuda")
        if B * H * lists.shape[2] > 30000:
            return None
        for b in range(B):
            at = torch.arange(ends[b], device="cuda")
            for h in range(H):
                kh, vh = k[b, :, h // shared].to(F64), vt[b, h // shared * D : (h // shared + 1) * D].to(F64).t().contiguous()
                for n, row in enumerate(lists[b, h].tolist()):
                    keys = torch.cat([at[KB * i : KB * i + KB] for i in row if i >= 0] or [at[:0]])
                    if len(keys):
                        p = torch.softmax(q[b, QB * n : QB * n + QB, h].to(F64) @ kh[keys].t() * SCALE, 1)
                        out[b, QB * n : QB * n + QB, h] = p @ vh[keys]
        return out
    if s["op"] == "quantise":
        return _round4(s["x"])
    M, K, N = case["M"], case["K"], case["N"]
    low, high = s["codes"].to(torch.int64) & 15, s["codes"].to(torch.int64) >> 4
    r, j = torch.meshgrid(torch.arange(N, device="cuda"), torch.arange(K // 32, device="cuda"), indexing="ij")
    tile = (r // 128) * ((K + 255) // 256) + j // 8
    e = s["scales"][tile * 1024 + (j % 4) * 256 + (r % 128 // 8) * 16 + (j % 8 // 4) * 8 + r % 8].to(F64) - 127
    w = torch.empty(N, K, dtype=F64, device="cuda")
    for part, c in ((0, low), (1, high)):
        ex, mant = (c >> 1) & 3, (c & 1).to(F64)                                # sign, two bits of exponent (bias 1), one of mantissa
        w[:, part::2] = torch.where(c >= 8, -1.0, 1.0) * torch.where(ex > 0, (1 + mant / 2) * 2.0 ** (ex - 1).to(F64), mant / 2)
    w = (w.view(N, K // 32, 32) * 2.0 ** e.unsqueeze(2)).view(N, K)
    y = _round4(s["x"]) @ w.t() + s["bias"].to(F64)
    if case["epilogue"] == "gelu":
        return y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if case["epilogue"] == "gate":
        return s["residual"].to(F64) + y * (s["mod"][GATE].to(F64) + s["e"][0, GATE].to(F64))
    if case["epilogue"] == "transposed":
        return torch.nn.functional.pad(y.t(), (0, -M % 64))
    return y
