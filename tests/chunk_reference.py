"""Attention of new tokens over a paged cache in 64 bits, the error bound of the kernels, and seeded batches (on any device)."""

import math

import torch


def make_chunk_case(seed, new, lens, hq, hkv, d, tpp=16, dtype=torch.bfloat16, device="cpu", window=None, q_scale=1.0, extra_rows=0,
                    poison=True):
    """A batch whose pools hold NaN everywhere but in the keys that some row may see, and whose page table holds garbage
    wherever no such key lies."""
    g = torch.Generator().manual_seed(seed)
    S = len(new)
    counts = [-(-max(L, 0) // tpp) for L in lens]
    total = max(sum(counts) + 2, 1)
    perm = torch.randperm(total, generator=g)
    table = torch.full((S, max(counts + [1]) + 1), -1, dtype=torch.int64)
    k = torch.full((total, tpp, hkv, d), float("nan") if poison else 0.5).to(dtype)
    v = torch.full((total, tpp, hkv, d), float("nan") if poison else 0.5).to(dtype)
    at = 0
    for s, (n, L, c) in enumerate(zip(new, lens, counts)):
        ids = perm[at:at + c]
        at += c
        lowest = max(0, L - n - window + 1) if window else 0
        if L > 0:
            tok = torch.arange(lowest, L)
            k[ids[tok // tpp], tok % tpp] = torch.randn((len(tok), hkv, d), generator=g).to(dtype)
            v[ids[tok // tpp], tok % tpp] = torch.randn((len(tok), hkv, d), generator=g).to(dtype)
        table[s, lowest // tpp:c] = ids[lowest // tpp:]
    q = (torch.randn((sum(new) + extra_rows, hq, d), generator=g) * q_scale).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0))) if S else torch.zeros(1)
    to = lambda t: t.contiguous().to(device)
    return dict(q=to(q), k_pool=to(k.view(total, tpp, hkv, d // 8, 8).permute(0, 2, 3, 1, 4)), v_pool=to(v.permute(0, 2, 3, 1)),
                table=to(table.to(torch.int32)), lens=to(torch.tensor(lens, dtype=torch.int32)), cu=to(cu.to(torch.int32)), new=list(new),
                lens_list=list(lens), window=window)


def chunk_reference(case, causal=True, scale=None):
    """(out, bound): float64 outputs [T, Hq, D] and the largest error of a kernel with fp32 accumulation, rows of no sequence 0.

    The bound, per output element with weights p over n keys, A = sum p |v| and B = sum |v|:
      * a score is a sum of D products in fp32, off by at most delta = D 2^-24 sum |q k| scale, and the exponential by 2^-22:
        weights off by a relative 2 delta + 2^-22, the output by that times (A + |out|);
      * sums over n keys in fp32: n 2^-24 A;
      * P rounded to 16 bits: half a step, eps / 2, of every weight: eps / 2 A, and below fp16's normal range half its smallest
        step, 2^-25 of the largest weight or less: 2^-25 B (numerator scaled so that the denominator is at least 1).
    The rounding of the output comes on top (see assert_chunk)."""
    q, kp, vp, table = case["q"], case["k_pool"], case["v_pool"], case["table"]
    total_pages, hkv, d, tpp = vp.shape
    hq = q.shape[1]
    group = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    eps = torch.finfo(q.dtype).eps
    row = 0
    for s, (n, L) in enumerate(zip(case["new"], case["lens_list"])):
        if n and L > 0:
            tok = torch.arange(L, device=q.device)
            pos = torch.arange(L - n, L, device=q.device)
            seen = tok[None] <= (pos[:, None] if causal else L - 1)
            if case["window"]:
                seen = seen & (tok[None] > pos[:, None] - case["window"])
            used = seen.any(0)
            page = table[s].long()[torch.where(used, tok // tpp, 0)].clamp(0, total_pages - 1)
            zero = torch.zeros((), dtype=torch.float64, device=q.device)
            k = torch.where(used[:, None, None], kp[page, :, :, tok % tpp].reshape(L, hkv, d).double(), zero)
            v = torch.where(used[:, None, None], vp[page, :, :, tok % tpp].double(), zero)
            for h in range(hkv):
                qh = q[row:row + n, h * group:(h + 1) * group].double()  # [n, G, D]
                score = torch.einsum("ngd,ld->ngl", qh, k[:, h]) * scale
                score = score.masked_fill(~seen[:, None], -math.inf)
                top = score.amax(-1, keepdim=True)
                top = torch.where(top == -math.inf, zero, top)
                w = torch.exp(score - top)
                total = w.sum(-1, keepdim=True)
                p = torch.where(total > 0, w / total, zero)
                o = torch.einsum("ngl,ld->ngd", p, v[:, h])
                A = torch.einsum("ngl,ld->ngd", p, v[:, h].abs())
                Bsum = torch.einsum("nl,ld->nd", seen.double(), v[:, h].abs())[:, None]
                size = torch.einsum("ngd,ld->ngl", qh.abs(), k[:, h].abs()).masked_fill(~seen[:, None], 0).amax(-1, keepdim=True) * scale
                delta = d * 2.0 ** -24 * size
                keys = seen.sum(-1).double()[:, None, None]
                b = (2 * delta + 2.0 ** -22) * (A + o.abs()) + keys * 2.0 ** -24 * A
                b = b + eps / 2 * A + (2.0 ** -25 * Bsum if q.dtype == torch.float16 else 0)
                out[row:row + n, h * group:(h + 1) * group] = o
                bound[row:row + n, h * group:(h + 1) * group] = b
        row += n
    return out, bound


def assert_chunk(got, case, causal=True, scale=None):
    ref, bound = chunk_reference(case, causal, scale)
    rows = sum(case["new"])
    got = got[:rows].double()
    ref, bound = ref[:rows], bound[:rows]
    assert torch.isfinite(got).all(), "non-finite values in the output"
    if case.get("out_dtype") != torch.float32:
        info = torch.finfo(case["q"].dtype)
        bound = bound + info.eps / 2 * (ref.abs() + bound) + (2.0 ** -25 if case["q"].dtype == torch.float16 else 0)
    excess = ((got - ref).abs() - bound)
    worst = excess.max().item() if excess.numel() else 0.0
    assert worst <= 0, f"largest error past the bound {worst:.3e} at {(excess == excess.max()).nonzero()[0].tolist()}"
